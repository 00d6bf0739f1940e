// Low-rank adapters on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// lora_tile_kernel: two chained products for a tile of 128 rows of one adapter,
//   DIR 0, forward:   u = x A^T [128, R]       out = base + (s u) B^T
//   DIR 1, gradient:  v = s dy B [128, R]      dx  = base + v A
// by a thread-block cluster of C CTAs.  CTA c sums a slice of the long first
// contraction (H or N); the partial [128, R] sums meet in fp32 through
// distributed shared memory, and CTA c computes a slice of the output columns.
// The work is bound by HBM: rows in, base in, rows out, each once.
//
// lora_dw_kernel: dA^T [H, R] = x^T v and dB [N, R] = s dy^T u, the rows of the
// adapter as the contraction, one tile of 128 columns of x or dy per cluster,
// whose CTAs share the rows; partial sums meet the same way, in rank order.
//
// Precision: x, dy, A and B are BF16 as given.  u and v are fp32 sums; as
// operands of the second product they are carried as two BF16 values each
// (hi = bf16(u), lo = bf16(u - hi)), an error of 2^-16 instead of 2^-8: the
// second product costs twice the MMAs, which HBM hides, and the output has one
// visible rounding.
//
// Operands come in by cp.async (rows are gathered by token, 16 bytes a lane)
// into 128-byte-swizzled tiles, kStages deep.  Every column beyond an
// adapter's rank, every row beyond a tile and every column beyond a matrix is
// filled with zeros there, whatever memory holds.  One thread issues the MMAs;
// all threads load and drain, one __syncthreads per step.  Two CTAs fit an SM
// (R <= 64), so that one loads while the other drains.
//
// Waits for MMAs are bounded: on a timeout the CTA sets the device error word
// (zmoe_kernel_error), stops waiting and runs through to its end, so that no
// CTA of its cluster is left at a barrier; its outputs are then incomplete.
#include <cooperative_groups.h>

#include "lora.cuh"
#include "tc.cuh"

namespace cg = cooperative_groups;

namespace zmoe {
namespace lora {

__device__ int32_t g_lora_error = 0;

namespace {

using namespace tc;

constexpr int kTile = 128;                             // rows per tile (MMA M)
constexpr int kStep = 64;                              // contraction or output columns per step: 128 bytes
constexpr int kStages = 3;
constexpr int kXBytes = kTile * kStep * 2;             // 16 KB
constexpr uint32_t kTmemCols = 256;                    // [0, 128): first product, [128, 256): two 64-column outputs
constexpr long long kWaitLimit = 4000000000LL;         // about 2 s at 1.9 GHz

// fp32 D, BF16 A and B, M = 128; amn / bmn: the operand's M or N index is contiguous
__device__ __forceinline__ uint32_t idesc(int n, int amn, int bmn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)amn << 15) | ((uint32_t)bmn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// Operand whose M or N index is contiguous, 128-byte swizzle: 64 of them per
// 128-byte row, one row per contraction index; 8 rows (1024 bytes) to the next
// group of contraction indices, 64-wide blocks `block` bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t block) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// 16-byte asynchronous copy of the first `bytes` (0..16) of src, zeros behind them.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&f)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r[i]);
}

// Bounded; after the first timeout the CTA no longer waits.
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (!mbar_try_wait(bar, parity)) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
      if (*failed) break;
      if (clock64() - t0 > kWaitLimit) {
        *failed = 1;
        atomicExch(&g_lora_error, 1);
        break;
      }
    }
  }
  __syncwarp();
}

// 16-byte place (row, chunk of 8 columns) of a 128-byte-swizzled tile of 64-column blocks.
__device__ __forceinline__ uint32_t place(int row, int chunk, uint32_t block) {
  return (uint32_t)(chunk >> 3) * block + (uint32_t)row * 128u + (uint32_t)(((chunk & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_bf16_bits(a) | ((uint32_t)f32_to_bf16_bits(b) << 16);
}

// Eight fp32 values as two BF16 vectors, f = hi + lo up to 2^-16; an infinite
// hi has no remainder.
__device__ __forceinline__ void split8(const float (&f)[8], uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float v = f[2 * q + i], b = round_bf16(v);
      r[i] = fabsf(b) <= 3.4e38f ? v - b : 0.0f;
    }
    h[q] = pack2(f[2 * q], f[2 * q + 1]);
    l[q] = pack2(r[0], r[1]);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

struct TileArgs {
  const uint16_t* src;                                 // [T, K1] rows of the first product
  const uint16_t* w1;                                  // DIR 0: A [G, R, K1]; DIR 1: B [G, K1, R]
  const uint16_t* w2;                                  // DIR 0: B [G, K2, R]; DIR 1: A [G, R, K2]
  const uint16_t* base;                                // [T, K2] or nullptr
  const float* scale;
  const int32_t *rank, *offsets, *token_of_row;
  int T, K1, K2, G, R;
  uint16_t* out;                                       // [T, K2] or nullptr (DIR 1: only v)
  float* u;                                            // [T, R] or nullptr: u (DIR 0) or s dy B (DIR 1)
};

__device__ __forceinline__ int rank_of(const int32_t* rank, int g, int R) {
  return rank ? min(max(rank[g], 0), R) : R;
}

// RB: 64-wide blocks of the rank (R <= 64 * RB).
template <int RB>
constexpr int tile_smem() { return 1024 + kStages * (kXBytes + RB * 8192) + RB * 2 * 16384; }

template <int DIR, int RB>
__global__ void __launch_bounds__(kThreads, RB == 1 ? 2 : 1) lora_tile_kernel(const TileArgs a) {
  constexpr uint32_t kWBytes = RB * 8192, kStageBytes = kXBytes + kWBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar[kStages];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ Unit unit_s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int q = warp & 3, half = warp >> 2;            // TMEM lane quarter and column half of this warp
  if (warp == 0) {
    const Unit u = find_unit(a.offsets, a.G, a.T, kTile, a.out && a.out != a.base, (int)(blockIdx.x / csize));
    if (lane == 0) unit_s = u;
  }
  __syncthreads();
  const Unit un = unit_s;
  if (un.rows == 0) return;                            // the whole cluster leaves
  const int K1 = a.K1, K2 = a.K2, R = a.R, g = un.g;
  const int rk = g < a.G ? rank_of(a.rank, g, R) : 0;

  // this thread's chunk and its four rows of every 128 x 64 tile: a warp fills
  // and drains the same 32 rows x 32 columns
  const int c8 = half * 4 + (lane & 3);
  int tok[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = q * 32 + (lane >> 2) + 8 * j;
    tok[j] = m < un.rows ? token_of(a.token_of_row, un.row0 + m, a.T) : -1;
  }
  // output columns of this CTA, in steps
  const int c_all = a.out ? (K2 + kStep - 1) / kStep : 0, c_per = (c_all + csize - 1) / csize;
  const int cb = min(c_all, rank * c_per), nc = min(c_all, cb + c_per) - cb;

  if (rk == 0) {                                       // no adapter: out = base
    if (a.u && g < a.G)
      for (int i = rank * kThreads + tid; i < un.rows * R; i += csize * kThreads) a.u[(size_t)un.row0 * R + i] = 0.f;
    if (a.out == a.base) return;
    for (int s = 0; s < nc; ++s) {
      const int col = (cb + s) * kStep + 8 * c8;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (tok[j] >= 0 && col < K2) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (a.base) v = *reinterpret_cast<const uint4*>(a.base + (size_t)tok[j] * K2 + col);
          *reinterpret_cast<uint4*>(a.out + (size_t)tok[j] * K2 + col) = v;
        }
    }
    return;
  }

  const int rp = (rk + 15) & ~15;                      // the MMAs' N of the first product, K of the second
  const float scale = a.scale ? a.scale[g] : 1.0f;
  const int k_all = (K1 + kStep - 1) / kStep, k_per = (k_all + csize - 1) / csize;
  const int kb = min(k_all, rank * k_per), nk = min(k_all, kb + k_per) - kb;
  const int total = nk + nc;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ub = smem + kStages * kStageBytes;          // hi blocks, lo blocks; before that the partial sums
  float* part = reinterpret_cast<float*>(ub);          // [rp][kTile]
  const uint32_t ring = smem_u32(smem), ua = smem_u32(ub);

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // rows of the rank, 64 columns from col0 on: A's
  auto load_rank_rows = [&](uint32_t dst, const uint16_t* w, int K, int col0) {
    for (int i = tid; i < rp * 8; i += kThreads) {
      const int r = i >> 3, c = i & 7, col = col0 + 8 * c;
      const bool in = r < rk && col < K;
      cp16(dst + place(r, c, 0), in ? w + ((size_t)g * R + r) * K + col : w, in ? 16 : 0);
    }
  };
  // 64 rows from row0 on, columns of the rank: B's
  auto load_rank_cols = [&](uint32_t dst, const uint16_t* w, int K, int row0) {
    const int n8 = rp / 8;
    for (int i = tid; i < 64 * n8; i += kThreads) {
      const int n = i / n8, c = i - n * n8;
      const int bytes = row0 + n < K ? min(max(2 * (rk - 8 * c), 0), 16) : 0;
      cp16(dst + place(n, c, 8192), bytes ? w + ((size_t)g * K + row0 + n) * R + 8 * c : w, bytes);
    }
  };
  auto load = [&](int s) {
    if (s < total) {
      const uint32_t st = ring + (uint32_t)(s % kStages) * kStageBytes;
      const bool first = s < nk;
      const uint16_t* rows = first ? a.src : a.base;
      const int K = first ? K1 : K2;
      const int col0 = (first ? kb + s : cb + s - nk) * kStep, col = col0 + 8 * c8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = rows && tok[j] >= 0 && col < K;
        cp16(st + place(q * 32 + (lane >> 2) + 8 * j, c8, 0), in ? rows + (size_t)tok[j] * K + col : a.src, in ? 16 : 0);
      }
      if (first == (DIR == 0)) load_rank_rows(st + kXBytes, first ? a.w1 : a.w2, K, col0);
      else load_rank_cols(st + kXBytes, first ? a.w1 : a.w2, K, col0);
    }
    cp_commit();
  };

  load(0);
  load(1);
  for (int s = 0; s <= total; ++s) {
    cp_wait<1>();                                      // this thread's copies of step s have landed
    if (s == nk) {
      // ---- the partial sums of the cluster become the second product's operand --------
      if (nk > 0) wait_bar(&bar[(nk - 1) % kStages], (uint32_t)((nk - 1) / kStages) & 1u, &failed);
      tc_fence_after();
      float f[RB * 4][8];
#pragma unroll
      for (int i = 0; i < RB * 4; ++i) {
        const int c0 = half * (rp / 2) + 8 * i;
        if (8 * i < rp / 2) {
          if (nk > 0) {
            tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0, f[i]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] = 0.0f;
          }
          if (csize > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) part[(c0 + e) * kTile + q * 32 + lane] = f[i][e];
          }
        }
      }
      if (csize > 1) {
        cl.sync();
#pragma unroll
        for (int i = 0; i < RB * 4; ++i) {
          const int c0 = half * (rp / 2) + 8 * i;
          if (8 * i < rp / 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] = 0.0f;
            for (int c = 0; c < csize; ++c) {
              const float* p = cl.map_shared_rank(part, c) + c0 * kTile + q * 32 + lane;
#pragma unroll
              for (int e = 0; e < 8; ++e) f[i][e] += p[e * kTile];
            }
          }
        }
        cl.sync();                                     // every CTA has read; the operand takes the place
      }
      const int m = q * 32 + lane;
      float* urow = a.u && rank == 0 && m < un.rows ? a.u + (size_t)(un.row0 + m) * R : nullptr;
#pragma unroll
      for (int i = 0; i < RB * 4; ++i) {
        const int c0 = half * (rp / 2) + 8 * i;
        if (8 * i < rp / 2) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (c0 + e >= rk) f[i][e] = 0.0f;
            v[e] = f[i][e] * scale;
          }
          if (urow && c0 < R) {
            float4* up = reinterpret_cast<float4*>(urow + c0);
            up[0] = DIR ? make_float4(v[0], v[1], v[2], v[3]) : make_float4(f[i][0], f[i][1], f[i][2], f[i][3]);
            up[1] = DIR ? make_float4(v[4], v[5], v[6], v[7]) : make_float4(f[i][4], f[i][5], f[i][6], f[i][7]);
          }
          uint4 hi, lo;
          split8(v, hi, lo);
          const uint32_t o = place(m, c0 / 8, 16384);
          *reinterpret_cast<uint4*>(ub + o) = hi;
          *reinterpret_cast<uint4*>(ub + RB * 16384 + o) = lo;
        }
      }
      if (urow && half == 0)
        for (int c = rp; c < R; c += 4) *reinterpret_cast<float4*>(urow + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    fence_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && s < total) {
      const uint32_t st = ring + (uint32_t)(s % kStages) * kStageBytes, w = st + kXBytes;
      if (s < nk) {
        const uint32_t id = idesc(rp, 0, DIR);
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk)
          tc_mma(tmem, smem_desc(st) + 2 * kk, DIR ? desc_mn(w + 2048 * kk, 8192) : smem_desc(w) + 2 * kk, id,
                 (s | kk) != 0);
      } else {
        const uint32_t id = idesc(kStep, 0, DIR), d = tmem + 128 + 64 * (uint32_t)((s - nk) & 1);
        for (int kk = 0; kk < rp / 16; ++kk) {
          const uint64_t db = DIR ? desc_mn(w + 2048 * kk, 8192) : smem_desc(w + (kk >> 2) * 8192) + 2 * (kk & 3);
          const uint64_t dh = smem_desc(ua + (kk >> 2) * 16384) + 2 * (kk & 3);
          const uint64_t dl = smem_desc(ua + RB * 16384 + (kk >> 2) * 16384) + 2 * (kk & 3);
          tc_mma(d, dh, db, id, kk != 0);
          tc_mma(d, dl, db, id, 1);
        }
      }
      tc_commit(&bar[s % kStages]);
    }
    __syncwarp();
    if (s > 0) wait_bar(&bar[(s - 1) % kStages], (uint32_t)((s - 1) / kStages) & 1u, &failed);
    if (s > nk) {
      // ---- drain the output of step s - 1: base plus product, one rounding -------------
      const int o = s - 1 - nk;
      uint8_t* xt = smem + (size_t)((s - 1) % kStages) * kStageBytes;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float d[8], b[8];
        tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + 128u + 64u * (uint32_t)(o & 1) + (uint32_t)(half * 32 + 8 * c), d);
        uint4* p = reinterpret_cast<uint4*>(xt + place(q * 32 + lane, half * 4 + c, 0));
        unpack8(*p, b);
        *p = make_uint4(pack2(b[0] + d[0], b[1] + d[1]), pack2(b[2] + d[2], b[3] + d[3]),
                        pack2(b[4] + d[4], b[5] + d[5]), pack2(b[6] + d[6], b[7] + d[7]));
      }
      __syncwarp();
      const int col = (cb + o) * kStep + 8 * c8;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (tok[j] >= 0 && col < K2)
          *reinterpret_cast<uint4*>(a.out + (size_t)tok[j] * K2 + col) =
              *reinterpret_cast<const uint4*>(xt + place(q * 32 + (lane >> 2) + 8 * j, c8, 0));
      __syncwarp();
    }
    load(s + 2);
  }
  cp_wait<0>();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------------
// dA and dB
// ---------------------------------------------------------------------------
struct DwArgs {
  const uint16_t* src[2];                              // x [T, H], dy [T, N]
  const float* f[2];                                   // v [T, R], u [T, R]
  uint16_t* out[2];                                    // da [G, R, H], db [G, N, R]
  const float* scale;
  const int32_t *rank, *offsets, *token_of_row;
  int M[2];                                            // H, N
  int T, G, R;
};

template <int RB>
constexpr int dw_smem() { return 1024 + kStages * (kXBytes + RB * 2 * 8192); }

template <int RB>
__global__ void __launch_bounds__(kThreads, RB == 1 ? 2 : 1) lora_dw_kernel(const DwArgs a) {
  constexpr uint32_t kStageBytes = kXBytes + RB * 2 * 8192;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar[kStages];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = warp & 3, half = warp >> 2;
  const int tilesA = (a.M[0] + kTile - 1) / kTile;
  const int unit = (int)(blockIdx.x / csize), g = blockIdx.y;
  const int which = unit >= tilesA, m0 = (which ? unit - tilesA : unit) * kTile, M = a.M[which];
  const int R = a.R, rk = rank_of(a.rank, g, R);
  const int r0 = min(max(a.offsets[g], 0), a.T), r1 = min(max(a.offsets[g + 1], 0), a.T);
  uint16_t* out = a.out[which];
  const int m = m0 + q * 32 + lane;                    // this thread's column of src (TMEM lane)

  // eight rank columns from c0 on of column m
  auto store = [&](int c0, const float (&v)[8]) {
    if (m >= M || c0 >= R) return;
    if (which) {
      *reinterpret_cast<uint4*>(out + ((size_t)g * M + m) * R + c0) =
          make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[((size_t)g * R + c0 + e) * M + m] = f32_to_bf16_bits(v[e]);
    }
  };
  const float zero8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int rp = r1 > r0 ? (rk + 15) & ~15 : 0;
  for (int c = rp / 8 + rank * 2 + half; c < R / 8; c += 2 * csize) store(8 * c, zero8);
  if (rp == 0) return;                                 // the whole cluster leaves

  const int s_all = (r1 - r0 + kStep - 1) / kStep, s_per = (s_all + csize - 1) / csize;
  const int sb = min(s_all, rank * s_per), ns = min(s_all, sb + s_per) - sb;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem);
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(128)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // 64 rows x 128 columns of src per step: this thread's chunk and four rows
  const int ch = tid & 15, col = m0 + 8 * ch;
  const uint16_t* src = a.src[which];
  const float* fsrc = a.f[which];
  int tok[4];                                          // rows of the next load
  auto load_tok = [&](int s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = r0 + (sb + s) * kStep + (tid >> 4) + 16 * j;
      tok[j] = s < ns && row < r1 ? token_of(a.token_of_row, row, a.T) : -1;
    }
  };
  auto load_x = [&](int s) {
    if (s < ns) {
      const uint32_t st = ring + (uint32_t)(s % kStages) * kStageBytes;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = tok[j] >= 0 && col < M;
        cp16(st + place((tid >> 4) + 16 * j, ch, 8192), in ? src + (size_t)tok[j] * M + col : src, in ? 16 : 0);
      }
    }
    cp_commit();
  };
  // the factor's rows: 64 x rp fp32, eight columns per item
  const int n8 = rp / 8;
  float fr[RB * 2][8];
  auto load_f = [&](int s) {
#pragma unroll
    for (int i = 0; i < RB * 2; ++i) {
      const int it = tid + i * kThreads, kr = it / n8, c = it - kr * n8;
      const int row = r0 + (sb + s) * kStep + kr;
#pragma unroll
      for (int e = 0; e < 8; ++e) fr[i][e] = 0.0f;
      if (s < ns && kr < kStep && row < r1 && 8 * c < R &&
          (a.token_of_row == nullptr || (unsigned)__ldg(a.token_of_row + row) < (unsigned)a.T)) {
        const float4* p = reinterpret_cast<const float4*>(fsrc + (size_t)row * R + 8 * c);
        const float4 lo = __ldg(p), hi = __ldg(p + 1);
        const float t[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * c + e < rk) fr[i][e] = t[e];
      }
    }
  };
  auto store_f = [&](int s) {
    if (s >= ns) return;
    uint8_t* w = smem + (size_t)(s % kStages) * kStageBytes + kXBytes;
#pragma unroll
    for (int i = 0; i < RB * 2; ++i) {
      const int it = tid + i * kThreads, kr = it / n8, c = it - kr * n8;
      if (kr >= kStep) continue;
      uint4 hi, lo;
      split8(fr[i], hi, lo);
      const uint32_t o = place(kr, c, 8192);
      *reinterpret_cast<uint4*>(w + o) = hi;
      *reinterpret_cast<uint4*>(w + RB * 8192 + o) = lo;
    }
  };

  load_tok(0);
  load_x(0);
  load_tok(1);
  load_x(1);
  load_f(0);
  store_f(0);
  load_f(1);
  store_f(1);
  load_f(2);
  load_tok(2);
  for (int s = 0; s < ns; ++s) {
    cp_wait<1>();
    fence_async();
    __syncthreads();
    if (tid == 0) {
      const uint32_t st = ring + (uint32_t)(s % kStages) * kStageBytes, w = st + kXBytes;
      const uint32_t id = idesc(rp, 1, 1);
#pragma unroll
      for (int kk = 0; kk < kStep / 16; ++kk) {
        const uint64_t da = desc_mn(st + 2048 * kk, 8192);
        tc_mma(tmem, da, desc_mn(w + 2048 * kk, 8192), id, (s | kk) != 0);
        tc_mma(tmem, da, desc_mn(w + RB * 8192 + 2048 * kk, 8192), id, 1);
      }
      tc_commit(&bar[s % kStages]);
    }
    __syncwarp();
    if (s > 0) wait_bar(&bar[(s - 1) % kStages], (uint32_t)((s - 1) / kStages) & 1u, &failed);
    store_f(s + 2);
    load_x(s + 2);
    load_f(s + 3);
    load_tok(s + 3);
  }
  cp_wait<0>();
  if (ns > 0) wait_bar(&bar[(ns - 1) % kStages], (uint32_t)((ns - 1) / kStages) & 1u, &failed);
  tc_fence_after();
  __syncthreads();                                     // the ring is free: partial sums take its place
  float* part = reinterpret_cast<float*>(smem);        // [rp][kTile]
  const float scale = which && a.scale ? a.scale[g] : 1.0f;
  for (int c = half; c < n8; c += 2) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ns > 0) tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(8 * c), v);
    if (csize > 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) part[(8 * c + e) * kTile + q * 32 + lane] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * c + e < rk ? v[e] * scale : 0.0f;
      store(8 * c, v);
    }
  }
  if (csize > 1) {
    cl.sync();
    for (int c = rank * 2 + half; c < n8; c += 2 * csize) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int p = 0; p < csize; ++p) {
        const float* rp_ = cl.map_shared_rank(part, p) + 8 * c * kTile + q * 32 + lane;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += rp_[e * kTile];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * c + e < rk ? v[e] * scale : 0.0f;
      store(8 * c, v);
    }
    cl.sync();                                         // partial sums stay until every CTA has read them
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128) : "memory");
  }
}

template <class K, class A>
zmoe_status launch_clusters(K* kernel, dim3 grid, int csize, int smem, cudaStream_t stream, const A& args,
                            const char* what) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)csize;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, kernel, args));
  return launch_status(what);
}

// CTAs per cluster: enough that `units` clusters fill the SMs' two places, no
// more than there are steps to share.
int cluster_size(long long units, int steps, int per_sm) {
  int c = 1;
  while (c < 8 && 2 * c * units <= (long long)kNumSMs * per_sm && 2 * c <= steps) c *= 2;
  return c;
}

template <int DIR, int RB>
zmoe_status launch_tile(const TileArgs& a, cudaStream_t stream) {
  zmoe_status st = allow_smem<lora_tile_kernel<DIR, RB>>();
  if (st != ZMOE_OK) return st;
  const long long units = a.T / kTile + (a.T < a.G + 1 ? a.T : a.G + 1);
  const int csize = cluster_size(units, (a.K1 + kStep - 1) / kStep, RB == 1 ? 2 : 1);
  ZMOE_CHECK_ARG(units * csize < (1LL << 31), "lora: T=%d rows are too many for one launch", a.T);
  return launch_clusters(lora_tile_kernel<DIR, RB>, dim3((unsigned)(units * csize)), csize, tile_smem<RB>(), stream, a,
                         "lora_tile_kernel");
}

template <int RB>
zmoe_status launch_dw(const DwArgs& a, cudaStream_t stream) {
  zmoe_status st = allow_smem<lora_dw_kernel<RB>>();
  if (st != ZMOE_OK) return st;
  const int tiles = (a.M[0] + kTile - 1) / kTile + (a.M[1] + kTile - 1) / kTile;
  const int steps = (a.T + kStep - 1) / kStep;
  const int csize = cluster_size((long long)tiles * a.G, steps, RB == 1 ? 2 : 1);
  return launch_clusters(lora_dw_kernel<RB>, dim3((unsigned)(tiles * csize), (unsigned)a.G), csize, dw_smem<RB>(),
                         stream, a, "lora_dw_kernel");
}

}  // namespace

zmoe_status launch_tiles(const zmoe_lora_args* p, cudaStream_t stream) {
  const TileArgs a{p->x, p->a, p->b, p->base, p->scale, p->rank, p->offsets, p->token_of_row,
                   p->T, p->H, p->N, p->G, p->R, p->out, p->u};
  return p->R <= 64 ? launch_tile<0, 1>(a, stream) : launch_tile<0, 2>(a, stream);
}

zmoe_status launch_grad_tiles(const zmoe_lora_grad_args* p, cudaStream_t stream) {
  const TileArgs a{p->dy, p->b, p->a, p->base, p->scale, p->rank, p->offsets, p->token_of_row,
                   p->T, p->N, p->H, p->G, p->R, p->dx, p->v};
  zmoe_status st = p->R <= 64 ? launch_tile<1, 1>(a, stream) : launch_tile<1, 2>(a, stream);
  if (st != ZMOE_OK || !p->da) return st;
  const DwArgs d{{p->x, p->dy}, {p->v, p->u}, {p->da, p->db}, p->scale, p->rank, p->offsets, p->token_of_row,
                 {p->H, p->N}, p->T, p->G, p->R};
  return p->R <= 64 ? launch_dw<1>(d, stream) : launch_dw<2>(d, stream);
}

zmoe_status read_error(int32_t* out, int reset) {
  ZMOE_CUDA_RET(cudaMemcpyFromSymbol(out, g_lora_error, sizeof(int32_t)));
  if (reset) {
    const int32_t z = 0;
    ZMOE_CUDA_RET(cudaMemcpyToSymbol(g_lora_error, &z, sizeof(int32_t)));
  }
  return ZMOE_OK;
}

}  // namespace lora
}  // namespace zmoe
