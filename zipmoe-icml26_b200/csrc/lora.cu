// Low-rank adapters of many requests beside a shared projection.
//
//   u = x[t] A_g^T     out[t] = base[t] + s_g u B_g^T      (t in the rows of adapter g)
// A batch's rows are grouped by adapter (offsets, token_of_row).  u stays fp32
// from the first product to the second, and out is rounded once.
//
// lora_rows_kernel, for few rows: a unit is up to kRows rows of one adapter and
// one thread-block cluster of kCluster CTAs.  The unit is bound by reading A_g
// and B_g once, and by latency: CTA c takes a slice of H for the first product
// (each weight vector serves all the unit's rows), the partial sums meet
// through distributed shared memory, and CTA c takes a slice of N for the
// second.  One launch, no scratch, no wait on another cluster.
#include <cooperative_groups.h>

#include "lora.cuh"

namespace cg = cooperative_groups;

namespace zmoe {
namespace lora {
namespace {

constexpr int kRows = 8;
constexpr int kCluster = 8;
constexpr int kRowsMaxT = 256;                         // longer batches go to the tensor cores
constexpr int kRG = 4;                                 // rank rows per warp pass
constexpr int kPre = 8;                                // 16-byte vectors of B loaded ahead of the sums

__global__ void __launch_bounds__(kThreads)
lora_rows_kernel(const zmoe_lora_args a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ Unit unit_s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const Unit u = find_unit(a.offsets, a.G, a.T, kRows, a.out != a.base, (int)(blockIdx.x / csize));
    if (lane == 0) unit_s = u;
  }
  __syncthreads();
  const Unit un = unit_s;
  if (un.rows == 0) return;                            // the whole cluster leaves
  const int H = a.H, N = a.N, R = a.R, nm = un.rows;
  const int ns = slice8(N, csize), n0 = min(N, rank * ns), n1 = min(N, n0 + ns);
  int tok[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) tok[m] = m < nm ? token_of(a.token_of_row, un.row0 + m, a.T) : -1;
  int rk = 0;
  float scale = 1.0f;
  if (un.g < a.G) {
    rk = a.rank ? min(max(a.rank[un.g], 0), R) : R;
    if (a.scale) scale = a.scale[un.g];
  }
  if (rk == 0) {                                       // no adapter: out = base
    if (a.u && un.g < a.G)
      for (int i = rank * kThreads + threadIdx.x; i < nm * R; i += csize * kThreads) a.u[(size_t)un.row0 * R + i] = 0.f;
    if (a.out == a.base) return;
    for (int m = 0; m < nm; ++m)
      if (tok[m] >= 0)
        for (int n = n0 + 8 * threadIdx.x; n < n1; n += 8 * kThreads) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (a.base) v = *reinterpret_cast<const uint4*>(a.base + (size_t)tok[m] * N + n);
          *reinterpret_cast<uint4*>(a.out + (size_t)tok[m] * N + n) = v;
        }
    return;
  }

  // ---- u, this CTA's slice of H --------------------------------------------------
  const int hs = slice8(H, csize), h0 = min(H, rank * hs), hn = min(H, h0 + hs) - h0;
  float* up = smem;                                    // [kRows][R] partial sums, read by the cluster
  float* us = up + kRows * R;                          // [kRows][R] scaled sums
  float* xs = us + kRows * R;                          // [kRows][hs] in two planes (elements 0-3 and 4-7 of each 8)
  const uint16_t* A = a.a + ((size_t)un.g * R) * H + h0;
  const uint16_t* B = a.b + ((size_t)un.g * N) * R;
  for (int i = threadIdx.x; i < nm * (hn / 8); i += kThreads) {
    const int m = i / (hn / 8), c = i % (hn / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    const int t = token_of(a.token_of_row, un.row0 + m, a.T);
    if (t >= 0) v = *reinterpret_cast<const uint4*>(a.x + (size_t)t * H + h0 + 8 * c);
    float f[8];
    unpack8(v, f);
    float* xp = xs + (size_t)m * hs + 4 * c;
    *reinterpret_cast<float4*>(xp) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(xp + hs / 2) = make_float4(f[4], f[5], f[6], f[7]);
  }
  __syncthreads();
  for (int r0 = kRG * warp; r0 < R; r0 += kRG * (kThreads / 32)) {
    float acc[kRG][kRows];
#pragma unroll
    for (int q = 0; q < kRG; ++q)
#pragma unroll
      for (int m = 0; m < kRows; ++m) acc[q][m] = 0.0f;
    if (r0 < rk) {
      for (int c = lane; c < hn / 8; c += 32) {
        float w[kRG][8];
#pragma unroll
        for (int q = 0; q < kRG; ++q) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r0 + q < rk) v = __ldg(reinterpret_cast<const uint4*>(A + (size_t)(r0 + q) * H) + c);
          unpack8(v, w[q]);
        }
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
          if (m >= nm) break;
          const float4 lo = *reinterpret_cast<const float4*>(xs + (size_t)m * hs + 4 * c);
          const float4 hi = *reinterpret_cast<const float4*>(xs + (size_t)m * hs + hs / 2 + 4 * c);
          const float xf[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int q = 0; q < kRG; ++q)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[q][m] = fmaf(xf[i], w[q][i], acc[q][m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      if (m >= nm) break;
#pragma unroll
      for (int q = 0; q < kRG; ++q) {
        float s = acc[q][m];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
        if (lane == 0) up[m * R + r0 + q] = s;
      }
    }
  }
  // ---- the first vectors of this thread's row of B, while the cluster meets ---------
  const int kv = (rk + 7) / 8;
  uint4 pre[kPre];
  const int nfirst = n0 + threadIdx.x;
#pragma unroll
  for (int q = 0; q < kPre; ++q)
    if (q < kv && nfirst < n1) pre[q] = __ldg(reinterpret_cast<const uint4*>(B + (size_t)nfirst * R) + q);
  cl.sync();
  for (int i = threadIdx.x; i < nm * R; i += kThreads) {
    float s = 0.0f;
    for (int c = 0; c < csize; ++c) s += *cl.map_shared_rank(up + i, c);
    if (rank == 0 && a.u) a.u[(size_t)un.row0 * R + i] = s;
    us[i] = s * scale;
  }
  __syncthreads();
  // ---- this CTA's slice of N ----------------------------------------------------------
  for (int n = nfirst; n < n1; n += kThreads) {
    float acc[kRows];
#pragma unroll
    for (int m = 0; m < kRows; ++m)
      acc[m] = (a.base && m < nm && tok[m] >= 0) ? bf16_bits_to_f32(a.base[(size_t)tok[m] * N + n]) : 0.0f;
    float sum[kRows];
#pragma unroll
    for (int m = 0; m < kRows; ++m) sum[m] = 0.0f;
    auto add = [&](const uint4& v, int q) {
      float w[8];
      unpack8(v, w);
      if (8 * q + 8 > rk) {                            // columns from the rank on may hold anything
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (8 * q + i >= rk) w[i] = 0.0f;
      }
#pragma unroll
      for (int m = 0; m < kRows; ++m) {
        if (m >= nm) break;
        const float4 lo = *reinterpret_cast<const float4*>(us + m * R + 8 * q);
        const float4 hi = *reinterpret_cast<const float4*>(us + m * R + 8 * q + 4);
        sum[m] += lo.x * w[0] + lo.y * w[1] + lo.z * w[2] + lo.w * w[3] + hi.x * w[4] + hi.y * w[5] + hi.z * w[6] +
                  hi.w * w[7];
      }
    };
    if (n == nfirst) {
#pragma unroll
      for (int q = 0; q < kPre; ++q)
        if (q < kv) add(pre[q], q);
    } else {
#pragma unroll 4
      for (int q = 0; q < min(kv, kPre); ++q) add(__ldg(reinterpret_cast<const uint4*>(B + (size_t)n * R) + q), q);
    }
    for (int q = kPre; q < kv; ++q) add(__ldg(reinterpret_cast<const uint4*>(B + (size_t)n * R) + q), q);
#pragma unroll
    for (int m = 0; m < kRows; ++m)
      if (m < nm && tok[m] >= 0) a.out[(size_t)tok[m] * N + n] = f32_to_bf16_bits(acc[m] + sum[m]);
  }
  cl.sync();                                           // partial sums stay until every CTA has read them
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
  ZMOE_CHECK_ARG(a->x && a->a && a->b && a->offsets && a->out && a->scratch, "lora: null pointer");
  ZMOE_CHECK_ARG(aligned16(a->x) && aligned16(a->base) && aligned16(a->a) && aligned16(a->b) && aligned16(a->out) &&
                     aligned16(a->u) && aligned16(a->scratch), "lora: rows must be 16-byte aligned");
  ZMOE_CHECK_ARG(a->H <= kMaxCols && a->N <= kMaxCols, "lora: H=%d or N=%d above %d", a->H, a->N, kMaxCols);
  if (a->T > kRowsMaxT) return launch_tiles(a, stream);
  zmoe_status st = allow_smem<lora_rows_kernel>();
  if (st != ZMOE_OK) return st;
  const size_t units = (size_t)a->T / kRows + (size_t)(a->T < a->G + 1 ? a->T : a->G + 1);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * kCluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(float) * (2 * kRows * (size_t)a->R + kRows * (size_t)slice8(a->H, kCluster));
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, lora_rows_kernel, *a));
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
  return launch_grad_tiles(a, stream);
}

}  // namespace zmoe
