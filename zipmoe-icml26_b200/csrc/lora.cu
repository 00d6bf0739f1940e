// Low-rank adapters of many requests beside a shared projection: entry points
// and the kernel for few rows.
//
//   u = x[t] A_g^T     out[t] = base[t] + s_g u B_g^T      (t in the rows of adapter g)
// A batch's rows are grouped by adapter (offsets, token_of_row).  u stays fp32
// from the first product to the second, and out is rounded once.
//
// lora_rows_kernel: a unit is up to kRows rows of one adapter and one
// thread-block cluster of kCluster CTAs.  The unit is bound by reading A_g and
// B_g once, and by latency, so the weights are the long side of the matrix
// instructions and go from global memory straight into their registers: with
// the contraction index permuted alike on both sides, a lane's fragments of two
// m16n8k16 steps are 16 contiguous bytes of a weight row and of a token's row.
// (tcgen05 would pay a trip through shared memory and TMEM for 8 columns; fp32
// multiply-adds instead of matrix instructions took twice as long at rank 64.)
// CTA c takes a slice of H for the first product, the partial sums meet through
// distributed shared memory, and CTA c takes a slice of N for the second.
// Weights do not wait for sums: a warp's first rows of B are in flight while the
// cluster meets.  One launch, no scratch, no wait on another cluster.
#include <cooperative_groups.h>

#include "lora.cuh"

namespace cg = cooperative_groups;

namespace zmoe {
namespace lora {
namespace {

constexpr int kRows = 8;                               // the matrix instruction's N
constexpr int kCluster = 8;                            // at most
constexpr int kWarps = kThreads / 32;
constexpr int kMaxR = ZMOE_LORA_MAX_RANK;
constexpr int kPitch = kMaxR + 32;                     // BF16 of a row of u: two rows' 64 bytes on different banks

__device__ __forceinline__ void mma16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                           uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 contraction indices: a lane's 16 bytes of weight rows l / 4 and l / 4 + 8, and of column l / 4.
__device__ __forceinline__ void mma32(float (&d)[4], const uint4& lo, const uint4& hi, const uint4& x) {
  mma16n8k16(d, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
  mma16n8k16(d, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
}

__device__ __forceinline__ uint4 ld16(const uint16_t* p, bool in) {
  return in ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

// Zeroes the elements from `left` (< 8) on of eight BF16.
__device__ __forceinline__ uint4 keep(uint4 v, int left) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = left >= 2 * q + 2 ? w[q] : left == 2 * q + 1 ? w[q] & 0xffffu : 0u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// KB: 32-wide blocks of the rank (R <= 32 * KB).  The fewer, the more tiles of B are in
// flight beside s u (96 requests of rank 16 15.2 us with room for two blocks, 13.0 for one).
template <int KB>
__global__ void __launch_bounds__(kThreads, 2)
lora_rows_kernel(const zmoe_lora_args a) {
  __shared__ Unit unit_s;
  __shared__ float part[8 * kRows * 16];               // [parts of the slice][kRows][ranks]
  __shared__ float up[kRows * kMaxR];                  // the CTA's sums, read by the cluster
  __shared__ __align__(16) uint16_t us[3][kRows * kPitch];   // s u, in three terms
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane >> 2, quad = lane & 3;
  if (warp == 0) {
    const Unit u = find_unit(a.offsets, a.G, a.T, kRows, a.out != a.base, (int)(blockIdx.x / csize));
    if (lane == 0) unit_s = u;
  }
  __syncthreads();
  const Unit un = unit_s;
  if (un.rows == 0) return;                            // the whole cluster leaves
  const int H = a.H, N = a.N, R = a.R, nm = un.rows, g = un.g;
  const int hs = slice8(H, csize), h0 = min(H, rank * hs), h1 = min(H, h0 + hs);
  const int ns = slice8(N, csize), n0 = min(N, rank * ns), n1 = min(N, n0 + ns);
  const int tok = row < nm ? token_of(a.token_of_row, un.row0 + row, a.T) : -1;   // of this lane's column
  const unsigned named = __ballot_sync(kFull, tok >= 0);   // bit 4 m: row m has a token
  int rk = 0;
  float scale = 1.0f;
  if (g < a.G) {
    rk = a.rank ? min(max(__ldg(a.rank + g), 0), R) : R;
    if (a.scale) scale = __ldg(a.scale + g);
  }
  if (rk == 0) {                                       // no adapter: out = base
    if (a.u && g < a.G)
      for (int i = rank * kThreads + tid; i < nm * R; i += csize * kThreads) a.u[(size_t)un.row0 * R + i] = 0.f;
    if (a.out == a.base) return;
    for (int m = 0; m < nm; ++m) {
      const int t = token_of(a.token_of_row, un.row0 + m, a.T);
      if (t < 0) continue;
      for (int n = n0 + 8 * tid; n < n1; n += 8 * kThreads) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (a.base) v = *reinterpret_cast<const uint4*>(a.base + (size_t)t * N + n);
        *reinterpret_cast<uint4*>(a.out + (size_t)t * N + n) = v;
      }
    }
    return;
  }
  const uint16_t* A = a.a + (size_t)g * R * H;
  const uint16_t* B = a.b + (size_t)g * N * R;

  // ---- u, this CTA's slice of H: warps share it as tiles of 16 ranks x parts -----------
  const int mt = (R + 15) / 16, parts = mt > 4 ? 1 : mt > 2 ? 2 : mt > 1 ? 4 : 8;
  const int blocks = (h1 - h0 + 31) / 32, per = (blocks + parts - 1) / parts;
  if (warp < mt * parts) {
    const int t16 = warp / parts, p = warp % parts;
    const int k0 = h0 + 32 * p * per, k1 = min(h1, k0 + 32 * per);
    const int r = 16 * t16 + row;
    const uint16_t* lo_p = A + (size_t)r * H;
    const uint16_t* hi_p = lo_p + (size_t)8 * H;
    const uint16_t* x_p = a.x + (size_t)max(tok, 0) * H;
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kB = 4;                              // blocks in flight
    for (int k = k0; k < k1; k += 32 * kB) {
      uint4 lo[kB], hi[kB], x[kB];
#pragma unroll
      for (int i = 0; i < kB; ++i) {
        const int kk = k + 32 * i + 8 * quad;
        const bool in = kk < k1;
        lo[i] = ld16(lo_p + kk, in && r < R);
        hi[i] = ld16(hi_p + kk, in && r + 8 < R);
        x[i] = ld16(x_p + kk, in && tok >= 0);
      }
#pragma unroll
      for (int i = 0; i < kB; ++i) mma32(d, lo[i], hi[i], x[i]);
    }
    float* pp = part + p * kRows * 16 * mt + 16 * t16 + row;   // [p][token][rank]
    pp[(2 * quad) * 16 * mt] = d[0];
    pp[(2 * quad + 1) * 16 * mt] = d[1];
    pp[(2 * quad) * 16 * mt + 8] = d[2];
    pp[(2 * quad + 1) * 16 * mt + 8] = d[3];
  }
  for (int i = tid; i < kRows * kPitch; i += kThreads) us[0][i] = us[1][i] = us[2][i] = 0;
  // ---- this warp's first tiles of B's rows, while the cluster meets -----------------------
  // A tile is 16 output columns: a lane's 16 bytes of rows l / 4 and l / 4 + 8 per
  // 32 ranks, and base at its four results (two columns, two tokens).
  const int k32 = (rk + 31) / 32, tiles = (n1 - n0 + 15) / 16;
  int t2[2];                                           // this lane's two tokens: 2 quad, 2 quad + 1
#pragma unroll
  for (int j = 0; j < 2; ++j)
    t2[j] = 2 * quad + j < nm ? token_of(a.token_of_row, un.row0 + 2 * quad + j, a.T) : -1;
  struct TileRegs {
    uint4 lo[KB], hi[KB];
    uint16_t base[4];
  };
  constexpr int kPre = 4 / KB;                         // with s u in registers, as many as fit
  TileRegs pre[kPre];
  auto load_tile = [&](int tile, TileRegs& w) {
    const int n = n0 + 16 * tile + row;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int k = 32 * kb + 8 * quad;
      w.lo[kb] = ld16(B + (size_t)n * R + k, n < n1 && k < rk);
      w.hi[kb] = ld16(B + (size_t)(n + 8) * R + k, n + 8 < n1 && k < rk);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int t = t2[c & 1], nn = n + 8 * (c >> 1);
      w.base[c] = a.base && t >= 0 && nn < n1 ? a.base[(size_t)t * N + nn] : (uint16_t)0;
    }
  };
#pragma unroll
  for (int j = 0; j < kPre; ++j)
    if (warp + kWarps * j < tiles) load_tile(warp + kWarps * j, pre[j]);
  __syncthreads();
  for (int i = tid; i < kRows * 16 * mt; i += kThreads) {
    const int m = i / (16 * mt), r = i % (16 * mt);
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += part[p * kRows * 16 * mt + i];
    if (r < R) up[m * R + r] = s;
  }
  cl.sync();
  for (int i = tid; i < nm * R; i += kThreads) {
    float p[kCluster];
#pragma unroll
    for (int c = 0; c < kCluster; ++c) p[c] = c < csize ? *cl.map_shared_rank(up + i, c) : 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < kCluster; ++c) s += p[c];
    const int m = i / R, r = i - m * R;
    if (r >= rk || !(named >> (4 * m) & 1)) s = 0.0f;   // a row of no token has u = 0
    if (rank == 0 && a.u) a.u[(size_t)un.row0 * R + i] = s;
    s *= scale;
    uint32_t t[3];
    split(s, t);
#pragma unroll
    for (int q = 0; q < 3; ++q) us[q][m * kPitch + r] = (uint16_t)(t[q] >> 16);
  }
  cl.barrier_arrive();                                 // partial sums stay until every CTA has read them
  __syncthreads();
  // s u of this lane, the same for every tile of B.  (Read again for each tile, its
  // three terms made shared memory the bound: 96 requests 22.4 us against 18.2.)
  uint4 uf[KB][3];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int q = 0; q < 3; ++q) uf[kb][q] = *reinterpret_cast<const uint4*>(&us[q][row * kPitch + 32 * kb + 8 * quad]);
  // ---- this CTA's slice of N --------------------------------------------------------------
  for (int t0 = warp; t0 < tiles; t0 += kWarps * kPre) {
#pragma unroll
    for (int j = 0; j < kPre; ++j) {
      const int tile = t0 + kWarps * j;
      if (tile >= tiles) break;
      float d[2][4] = {};                              // sums of the first term and of the others
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {                // columns from the rank on may hold anything
        const int k = 32 * kb + 8 * quad;
        if (k < rk && k + 8 > rk) {
          pre[j].lo[kb] = keep(pre[j].lo[kb], rk - k);
          pre[j].hi[kb] = keep(pre[j].hi[kb], rk - k);
        }
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        if (kb >= k32) break;
#pragma unroll
        for (int q = 0; q < 3; ++q) mma32(d[q > 0], pre[j].lo[kb], pre[j].hi[kb], uf[kb][q]);
      }
      const int n = n0 + 16 * tile + row;
#pragma unroll
      for (int c = 0; c < 4; ++c) {                    // rows n and n + 8, the lane's two tokens
        const int t = t2[c & 1], nn = n + 8 * (c >> 1);
        if (t >= 0 && nn < n1) a.out[(size_t)t * N + nn] = f32_to_bf16_bits(bf16_bits_to_f32(pre[j].base[c]) + (d[0][c] + d[1][c]));
      }
      if (tile + kWarps * kPre < tiles) load_tile(tile + kWarps * kPre, pre[j]);
    }
  }
  cl.barrier_wait();
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace
}  // namespace lora

zmoe_status launch_lora(const zmoe_lora_args* a, cudaStream_t stream) {
  using namespace lora;
  ZMOE_CHECK_ARG(a && a->T >= 0 && a->G >= 1, "lora: null pointer, T < 0 or G < 1");
  ZMOE_CHECK_ARG(a->H > 0 && a->H % 8 == 0 && a->N > 0 && a->N % 8 == 0, "lora: H=%d and N=%d must be positive multiples of 8",
                 a->H, a->N);
  ZMOE_CHECK_ARG(a->R > 0 && a->R % 8 == 0 && a->R <= ZMOE_LORA_MAX_RANK, "lora: R=%d must be a multiple of 8 in [8, %d]",
                 a->R, ZMOE_LORA_MAX_RANK);
  if (a->T == 0) return ZMOE_OK;
  ZMOE_CHECK_ARG(a->x && a->a && a->b && a->offsets && a->out && (a->scratch || a->T <= ZMOE_LORA_ROWS),
                 "lora: null pointer");
  ZMOE_CHECK_ARG(aligned16(a->x) && aligned16(a->base) && aligned16(a->a) && aligned16(a->b) && aligned16(a->out) &&
                     aligned16(a->u) && aligned16(a->scratch), "lora: rows must be 16-byte aligned");
  ZMOE_CHECK_ARG(a->H <= kMaxCols && a->N <= kMaxCols, "lora: H=%d or N=%d above %d", a->H, a->N, kMaxCols);
  ZMOE_CHECK_ARG(a->T <= kMaxT, "lora: T=%d above %d", a->T, kMaxT);
  {
    const size_t T = a->T, H = a->H, N = a->N, G = a->G, R = a->R;
    const Span w[] = {{"out", a->out, 2 * T * N, "base"}, {"u", a->u, 4 * T * R}, {"scratch", a->scratch, 4 * T * R}};
    const Span r[] = {{"x", a->x, 2 * T * H}, {"base", a->base, 2 * T * N}, {"a", a->a, 2 * G * R * H}, {"b", a->b, 2 * G * N * R},
                      {"scale", a->scale, 4 * G}, {"rank", a->rank, 4 * G}, {"offsets", a->offsets, 4 * (G + 1)},
                      {"token_of_row", a->token_of_row, 4 * T}};
    const char *p, *q;
    ZMOE_CHECK_ARG(apart(w, r, &p, &q), "lora: %s must not overlap %s", p, q);
  }
  // Few rows for each adapter: the rows kernel; else tiles of 128.  Measured (us, rows
  // against tiles, 2048 in and out): 512 rows 10.0 and 11.9 with one adapter of rank
  // 64, 12.8 and 39 with 128 of rank 16; 1024 rows 14.9 and 14.3, 9.4 and 12.0 at
  // rank 16, 28.7 and 51 with 128 of rank 64; 2048 rows 26.1 and 16.8.
  if (a->T > 2 * ZMOE_LORA_ROWS || (a->T > ZMOE_LORA_ROWS && a->R > 32 && a->G < 32)) return launch_tiles(a, stream);
  // as many CTAs per unit as fit the SMs together, two on each
  const int about = (a->T + kRows - 1) / kRows + (a->T < a->G ? a->T : a->G) / 2;
  const int units = a->T / kRows + (a->T < a->G + 2 ? a->T : a->G + 2);
  int csize = kCluster;
  while (csize > 1 && about * csize > 2 * kNumSMs) csize /= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * csize));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)csize;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, a->R <= 32 ? lora_rows_kernel<1> : a->R <= 64 ? lora_rows_kernel<2> : lora_rows_kernel<4>, *a));
  return launch_status("lora_rows_kernel");
}

zmoe_status launch_lora_grad(const zmoe_lora_grad_args* a, cudaStream_t stream) {
  using namespace lora;
  ZMOE_CHECK_ARG(a && a->T >= 0 && a->G >= 1, "lora_grad: null pointer, T < 0 or G < 1");
  ZMOE_CHECK_ARG(a->H > 0 && a->H % 8 == 0 && a->N > 0 && a->N % 8 == 0,
                 "lora_grad: H=%d and N=%d must be positive multiples of 8", a->H, a->N);
  ZMOE_CHECK_ARG(a->H <= kMaxCols && a->N <= kMaxCols, "lora_grad: H=%d or N=%d above %d", a->H, a->N, kMaxCols);
  ZMOE_CHECK_ARG(a->R > 0 && a->R % 8 == 0 && a->R <= ZMOE_LORA_MAX_RANK,
                 "lora_grad: R=%d must be a multiple of 8 in [8, %d]", a->R, ZMOE_LORA_MAX_RANK);
  ZMOE_CHECK_ARG((a->da == nullptr) == (a->db == nullptr), "lora_grad: da and db go together");
  ZMOE_CHECK_ARG(a->dx || a->da, "lora_grad: no output");
  ZMOE_CHECK_ARG(a->G <= 65535, "lora_grad: G=%d above 65535", a->G);
  ZMOE_CHECK_ARG(a->T <= kMaxT, "lora_grad: T=%d above %d", a->T, kMaxT);
  if (a->T == 0) {
    if (a->da) {
      ZMOE_CUDA_RET(cudaMemsetAsync(a->da, 0, sizeof(uint16_t) * (size_t)a->G * a->R * a->H, stream));
      ZMOE_CUDA_RET(cudaMemsetAsync(a->db, 0, sizeof(uint16_t) * (size_t)a->G * a->R * a->N, stream));
    }
    return ZMOE_OK;
  }
  ZMOE_CHECK_ARG(a->dy && a->a && a->b && a->offsets && a->scratch && (!a->da || (a->x && a->u)), "lora_grad: null pointer");
  ZMOE_CHECK_ARG(aligned16(a->dy) && aligned16(a->x) && aligned16(a->u) && aligned16(a->a) && aligned16(a->b) &&
                     aligned16(a->base) && aligned16(a->dx) && aligned16(a->da) && aligned16(a->db) && aligned16(a->scratch),
                 "lora_grad: rows must be 16-byte aligned");
  // dA and dB read dy and x after dx is written
  ZMOE_CHECK_ARG(!a->dx || !a->da || (a->dx != a->dy && a->dx != a->x), "lora_grad: dx must not be dy or x");
  {
    // without dA and dB, x and u are not read, and dx may be dy: its rows are written
    // after the first product has read them all
    const size_t T = a->T, H = a->H, N = a->N, G = a->G, R = a->R;
    const void* base = a->dx ? a->base : nullptr;
    const Span w[] = {{"dx", a->dx, 2 * T * H, base == a->dx ? "base" : a->da ? "" : "dy"}, {"da", a->da, 2 * G * R * H},
                      {"db", a->db, 2 * G * N * R}, {"scratch", a->scratch, 4 * T * R}};
    const Span r[] = {{"dy", a->dy, 2 * T * N}, {"x", a->da ? a->x : nullptr, 2 * T * H}, {"u", a->da ? a->u : nullptr, 4 * T * R},
                      {"a", a->a, 2 * G * R * H}, {"b", a->b, 2 * G * N * R}, {"scale", a->scale, 4 * G},
                      {"rank", a->rank, 4 * G}, {"offsets", a->offsets, 4 * (G + 1)},
                      {"token_of_row", a->token_of_row, 4 * T}, {"base", base, 2 * T * H}};
    const char *p, *q;
    ZMOE_CHECK_ARG(apart(w, r, &p, &q), "lora_grad: %s must not overlap %s", p, q);
  }
  return launch_grad_tiles(a, stream);
}

}  // namespace zmoe
