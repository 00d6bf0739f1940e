// Low-rank adapters on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// Three kernels, each bound by HBM (their MMAs are narrow):
//   lora_shrink_kernel  u = x A^T (forward) or v = s dy B (gradient) for tiles of
//                       128 rows of one adapter.  A cluster of C CTAs splits the
//                       long contraction (H or N) of a tile; the partial
//                       [128, R] sums meet in fp32 through distributed shared
//                       memory, each CTA adding its share of the columns in rank
//                       order.
//   lora_expand_kernel  out = base + s u B^T or dx = base + v A: a CTA per (tile,
//                       share of the output columns).  Launched as a dependent of
//                       the shrink: it loads base and weights while that ends.
//   lora_dw_kernel      dA^T = x^T v and dB = s dy^T u: the rows of an adapter as
//                       the contraction, one tile of 256 columns of x or dy per
//                       cluster, whose CTAs share the rows.  dB needs nothing of
//                       the launches in front and runs beside them; dA waits for
//                       them.
// (A single kernel for shrink and expand, with u kept in TMEM, measured slower:
// 31.5 against 28 us for 8191 rows of 2048 in and out at rank 64, 25 against 17 us
// for 2047 rows of 2048 in and 5632 out at rank 16: tiles of whole rows leave SMs
// without work.)
//
// Precision: x, dy, A and B are BF16 as given.  u and v are fp32 sums, and enter
// the second product whole: as three BF16 terms of 8 bits each whose sum they are.
// That costs three times the MMAs, which HBM hides, and the output has one
// rounding.  (Two terms, 16 bits, saved MMAs and a third of the operand's shared
// memory, but moved the outputs four times as far from an fp32 product's as the order
// of its sums does.)
//
// Warps have roles: some load, some split, one issues the MMAs, some drain TMEM.  Operands
// come in by cp.async (rows are gathered by token, 16 bytes a lane) into
// 128-byte-swizzled tiles of a ring, whose slots pass from role to role by
// mbarriers, so that no step waits for the whole CTA.  Every column beyond an
// adapter's rank and every column beyond a matrix is filled with zeros there,
// whatever memory holds.  Two CTAs fit an SM (R <= 64).
//
// Every mbarrier wait is bounded: on a timeout the CTA sets the device error
// word (zmoe_kernel_error), stops waiting and runs through to its end, so that
// no CTA of its cluster is left at a barrier; its outputs are then incomplete.
// TMEM allocations wait for nothing but CTAs that end by themselves: shared
// memory admits no more CTAs of these kernels to an SM than its 512 columns hold.
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
constexpr int kXBytes = kTile * kStep * 2;             // 16 KB

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
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on bar once this thread's copies so far have landed.  The copies
// are ordinary writes to the tensor cores' asynchronous reads, so the MMA warp
// fences between its wait and its MMAs.
__device__ __forceinline__ void cp_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void st16(uint32_t dst, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The MMA warp runs its loop with all lanes, so that barrier addresses and
// descriptors stay in uniform registers; `go` is true in the one lane that issues.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)
      : "memory");
}

// The same with A in TMEM.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)
      : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t go;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(go));
  return go;
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint4& v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns, 16 at a time, one wait.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&lo)[16], uint32_t (&hi)[16]) {
  tmem_ld16(taddr, lo);
  tmem_ld16(taddr + 16, hi);
  tmem_wait_ld();
}

__device__ __forceinline__ bool try_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void commit_at(uint32_t bar, uint32_t go) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(go)
      : "memory");
}

// Place of a step in the ring: slot, and the parity of the slot's use.
template <int N>
struct Ring {
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// Waits are bounded: the first that runs out sets the CTA's flag and the device
// error word, and the CTA no longer waits.
struct Guard {
  volatile int* failed;
  long long limit;                                     // clock64 cycles
};
__device__ __forceinline__ void wait_one(uint32_t bar, uint32_t parity, const Guard& guard) {
  if (try_wait_at(bar, parity)) return;
  const long long t0 = clock64();
  while (!try_wait_at(bar, parity)) {
    if (*guard.failed) return;
    if (clock64() - t0 > guard.limit) {
      *guard.failed = 1;
      atomicExch(&g_lora_error, 1);
      return;
    }
  }
}
__device__ __forceinline__ void wait_bar(uint32_t bar, uint32_t parity, const Guard& guard) {
  wait_one(bar, parity, guard);
  __syncwarp();
}

// The MMA warp's last act: every MMA that it issued has finished (bounded, even
// after a wait has failed), so that TMEM and shared memory can go.
__device__ __forceinline__ void finish_mmas(uint64_t* bar, uint32_t go, long long limit) {
  commit_at(smem_u32(bar), go);
  const long long t0 = clock64();
  while (!try_wait_at(smem_u32(bar), 0) && clock64() - t0 < limit) {
  }
  __syncwarp();
}

// 16-byte place (row, chunk of 8 columns) of a 128-byte-swizzled tile of 64-column blocks.
__device__ __forceinline__ uint32_t place(int row, int chunk, uint32_t block) {
  return (uint32_t)(chunk >> 3) * block + (uint32_t)row * 128u + (uint32_t)(((chunk & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct TileArgs {
  const uint16_t* src;                                 // shrink: [T, K1]
  const uint16_t* w1;                                  // DIR 0: A [G, R, K1]; DIR 1: B [G, K1, R]
  const uint16_t* w2;                                  // DIR 0: B [G, K2, R]; DIR 1: A [G, R, K2]
  const uint16_t* base;                                // expand: [T, K2] or nullptr
  const float* scale;
  const int32_t *rank, *offsets, *token_of_row;
  int T, K1, K2, G, R;
  uint16_t* out;                                       // [T, K2]
  float* u;                                            // DIR 0: [T, R] out or nullptr
  float* second;                                       // factor of the second product, [T, R]: s u, or v
  long long weights;                                   // DIR 1: tiles of dB, 0 without
  int parts;                                           // expand: CTAs per tile
  long long limit;                                     // of a wait, in clock64 cycles
  int drop;                                            // error-path test: the loaders load nothing
};

__device__ __forceinline__ int rank_of(const int32_t* rank, int g, int R) {
  return rank ? min(max(__ldg(rank + g), 0), R) : R;
}

constexpr int kLoadWarps = 4, kLoaders = 32 * kLoadWarps;

// The places and sources of a loader thread's pieces of the weights, fixed but
// for a step's constant move: rows of the rank x 64 columns (A), or 64 rows x
// columns of the rank (B).
template <int RB, bool RANK_ROWS>
struct Weights {
  uint32_t at[RB * 4];                                 // place << 5 | bytes; 31: no piece
  int off[RB * 4];                                     // B: row * R + 8 chunk
  const uint16_t* p;
  const uint16_t* any;                                 // a valid address for pieces of no bytes
  size_t row16;                                        // A: 16 rows
  int left, col, K, R, rk, rp, lt;

  __device__ __forceinline__ Weights(const uint16_t* w, int g, int K_, int R_, int rk_, int rp_, int lt_, int step0)
      : any(w), K(K_), R(R_), rk(rk_), rp(rp_), lt(lt_) {
    col = step0 * kStep + 8 * (lt & 7);
    row16 = (size_t)16 * K;
    left = (K - step0 * kStep) * R;
    if (RANK_ROWS) {
      p = w + ((size_t)g * R + (lt >> 3)) * K + col;
    } else {
      p = w + ((size_t)g * K + step0 * kStep) * R;
      const int n8 = rp / 8;
      const uint32_t inv = (65536u + n8 - 1) / n8;     // exact for the indexes below 64 n8 <= 1024
#pragma unroll
      for (int i = 0; i < RB * 4; ++i) {
        const int it = lt + i * kLoaders, n = (int)((it * inv) >> 16), c = it - n * n8;
        at[i] = n < kStep ? place(n, c, 8192) << 5 | (uint32_t)min(max(2 * (rk - 8 * c), 0), 16) : 31u;
        off[i] = n * R + 8 * c;
      }
    }
  }
  // The pieces of this step into dst (and xo: place of row lt / 8, chunk lt % 8), then `steps` on.
  __device__ __forceinline__ void load(uint32_t dst, uint32_t xo, int steps) {
    if (RANK_ROWS) {
#pragma unroll
      for (int e = 0; e < RB * 4; ++e) {
        const int r = (lt >> 3) + 16 * e;
        if (r < rp) {
          const bool in = r < rk && col < K;
          cp16(dst + xo + 2048u * e, in ? p + e * row16 : any, in ? 16 : 0);
        }
      }
      p += steps * kStep;
      col += steps * kStep;
    } else {
#pragma unroll
      for (int e = 0; e < RB * 4; ++e) {
        if (at[e] != 31u) {
          const int bytes = off[e] < left ? (int)(at[e] & 31u) : 0;
          cp16(dst + (at[e] >> 5), bytes ? p + off[e] : any, bytes);
        }
      }
      p += (size_t)(steps * kStep) * R;
      left -= steps * kStep * R;
    }
  }
};

// Eight rows of a 128 x 64 tile of x or base: rows lt / 8 + 16 j, chunk lt % 8.
// Rows behind the tile's last repeat a token: an MMA row depends on its own row
// alone, and theirs are not written.
struct Rows {
  const uint16_t* p[8];
  const uint16_t* any;
  int col, K;
  bool none;

  __device__ __forceinline__ Rows(const uint16_t* rows, const uint16_t* any_, const int (&tok)[8], int K_, int lt, int step0)
      : any(any_), K(K_), none(rows == nullptr) {
    col = step0 * kStep + 8 * (lt & 7);
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = none ? any : rows + (size_t)(unsigned)tok[j] * (unsigned)K + col;
  }
  __device__ __forceinline__ void load(uint32_t dst, int steps) {
    if (!none && col - (col & (kStep - 1)) + kStep <= K) {   // all but a matrix's ragged last step
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cp16(dst + 2048u * j, p[j]);
        p[j] += steps * kStep;
      }
    } else {
      const int bytes = !none && col < K ? 16 : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) cp16(dst + 2048u * j, bytes ? p[j] : any, bytes);
    }
    col += steps * kStep;
  }
};

__device__ __forceinline__ void tile_tokens(int (&tok)[8], const TileArgs& a, const Unit& un, int lt) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    tok[j] = max(token_of(a.token_of_row, un.row0 + min((lt >> 3) + 16 * j, un.rows - 1), a.T), 0);
}

// ---------------------------------------------------------------------------
// first product
// ---------------------------------------------------------------------------
// RB: 64-wide blocks of the rank (R <= 64 * RB).
template <int RB>
struct Shrink {
  static constexpr uint32_t kStageBytes = kXBytes + RB * 8192;
  static constexpr int kPerSM = RB == 1 ? 2 : 1;
  static constexpr int kStages = RB == 1 ? 4 : 6;      // 96 KB / 192 KB
  static constexpr int kGroups = 2;                    // of loader warps, taking steps in turn
  static constexpr int kThreads = kGroups * kLoaders + 32;
  static constexpr int kSmem = 1024 + kStages * kStageBytes;
};

template <int DIR, int RB>
__global__ void __launch_bounds__(Shrink<RB>::kThreads, Shrink<RB>::kPerSM) lora_shrink_kernel(const TileArgs a) {
  using L = Shrink<RB>;
  constexpr int kStages = L::kStages, kTurn = L::kGroups, kMmaWarp = kTurn * kLoadWarps;
  constexpr uint32_t kSum = RB * 64, kTmemCols = 2 * kSum;   // two sums, of half the steps each
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], used[kStages], sums, last;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ Unit unit_s;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the expand's CTAs may come as SMs free up
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the token list, a share a CTA, and the ranks and scales come to L2 while the
  // unit is looked for, instead of one after the other behind it
  if (a.token_of_row)
    for (long long i = 32LL * (blockIdx.x * (long long)L::kThreads + tid); i < a.T; i += 32LL * gridDim.x * L::kThreads)
      prefetch(a.token_of_row + i);
  if (32 * tid < a.G) {
    if (a.rank) prefetch(a.rank + 32 * tid);
    if (a.scale) prefetch(a.scale + 32 * tid);
  }
  if (warp == 0) {
    const Unit u = find_unit(a.offsets, a.G, a.T, kTile, false, (int)((gridDim.x - 1 - blockIdx.x) / csize));
    if (lane == 0) unit_s = u;
  }
  if (warp == kMmaWarp) {                              // set up while the unit is looked for
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) {
        mbar_init(&full[s], kLoaders);
        mbar_init(&used[s], 1);
      }
      mbar_init(&sums, 1);
      mbar_init(&last, 1);
      failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto free_tmem = [&]() {
    if (warp == kMmaWarp)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  };
  const Unit un = unit_s;
  const Guard guard{&failed, a.limit};
  if (un.rows == 0) return free_tmem();                // the whole cluster leaves
  const int K1 = a.K1, R = a.R, g = un.g;
  const int lt = tid % kLoaders, group = tid / kLoaders;
  int tok[8];
  if (warp < kMmaWarp) tile_tokens(tok, a, un, lt);    // in flight with the rank and the scale
  const int rk = rank_of(a.rank, g, R);
  const float scale = a.scale ? __ldg(a.scale + g) : 1.0f;
  if (rk == 0) {
    if (DIR == 0 && a.u)
      for (int i = rank * L::kThreads + tid; i < un.rows * R; i += csize * L::kThreads) a.u[(size_t)un.row0 * R + i] = 0.f;
    return free_tmem();
  }
  const int rp = (rk + 15) & ~15;                      // the MMAs' N
  const int k_all = (K1 + kStep - 1) / kStep, k_per = (k_all + csize - 1) / csize;
  const int kb = min(k_all, rank * k_per), nk = min(k_all, kb + k_per) - kb;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem), full_a = smem_u32(full), used_a = smem_u32(used);

  if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ load
    const uint32_t xo = place(lt >> 3, lt & 7, 0);
    Rows rows(a.src, a.src, tok, K1, lt, kb + group);
    Weights<RB, DIR == 0> w(a.w1, g, K1, R, rk, rp, lt, kb + group);
    Ring<kStages> at;
    for (int e = 0; e < group; ++e) at.next();
    for (int s = group; s < nk && !a.drop; s += kTurn) {
      if (s >= kStages) wait_bar(used_a + 8 * at.slot, at.parity ^ 1u, guard);
      const uint32_t st = ring + at.slot * L::kStageBytes;
      rows.load(st + xo, kTurn);
      w.load(st + kXBytes, xo, kTurn);
      cp_arrive(full_a + 8 * at.slot);
#pragma unroll
      for (int e = 0; e < kTurn; ++e) at.next();
    }
    cp_wait_all();
  } else {
    // ------------------------------------------------------------------ MMAs
    // Its instructions are the step's critical path: descriptors are built once
    // and moved by additions.
    const uint32_t go = elect_one(), id = idesc(rp, 0, DIR);
    Ring<kStages> at;
    const uint64_t dx0 = smem_desc(ring);
    const uint64_t dw0 = DIR ? desc_mn(ring + kXBytes, 8192) : smem_desc(ring + kXBytes);
    constexpr uint32_t kPer = DIR ? 2048 >> 4 : 2;     // 16 contraction indices on in the weights
#pragma unroll 1
    for (int s = 0; s < nk; ++s) {
      wait_bar(full_a + 8 * at.slot, at.parity, guard);
      fence_async();
      const uint32_t off = at.slot * (L::kStageBytes >> 4);
#pragma unroll
      for (int kk = 0; kk < kStep / 16; ++kk) mma_ss(tmem + (kk & 1) * kSum, dx0 + off + 2 * kk, dw0 + off + kPer * kk, id, (s | kk >> 1) != 0, go);
      commit_at(used_a + 8 * at.slot, go);
      at.next();
    }
    commit_at(smem_u32(&sums), go);
    finish_mmas(&last, go, a.limit);
  }

  // ---- sums: this thread's row, eight rank columns at a time ---------------------------
  const int q = warp & 3, half = warp >> 2, m = q * 32 + lane, n8 = rp / 8;
  float4* part = reinterpret_cast<float4*>(smem);      // [rp / 4][kTile][4], in the ring's place
  const bool mine = m < un.rows && warp < kMmaWarp;
  const size_t grow = (size_t)(un.row0 + m);
  const bool named = mine && token_of(a.token_of_row, un.row0 + m, a.T) >= 0;   // a row of no token has u = 0
  auto write = [&](int i, float (&f)[8]) {
    const int c0 = 8 * i;
    if (!mine || c0 >= R) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!named || c0 + e >= rk) f[e] = 0.0f;
    if (DIR == 0 && a.u) {
      float4* up = reinterpret_cast<float4*>(a.u + grow * R + c0);
      up[0] = make_float4(f[0], f[1], f[2], f[3]);
      up[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= scale;
    float4* sp = reinterpret_cast<float4*>(a.second + grow * R + c0);
    sp[0] = make_float4(f[0], f[1], f[2], f[3]);
    sp[1] = make_float4(f[4], f[5], f[6], f[7]);
  };
  auto sums_of = [&](int i, float (&f)[8]) {
    const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(8 * i);
    uint32_t v[2][8];                                  // a tensor-core sum is cut, not rounded, at every MMA
    tmem_ld8(at, v[0]);
    tmem_ld8(at + kSum, v[1]);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[0][e]) + __uint_as_float(v[1][e]);
  };
  const int first = csize == 1 ? half : rank + csize * half, stride = 2 * csize;
  if (warp < kMmaWarp) wait_bar(smem_u32(&sums), 0, guard);   // every MMA has read the ring
  tc_fence_after();
  if (csize == 1) {
    if (warp < kMmaWarp)
      for (int i = first; i < n8; i += stride) {
        float f[8];
        sums_of(i, f);
        write(i, f);
      }
  } else {
    if (warp < kMmaWarp)
      for (int i = half; i < n8; i += 2) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (nk > 0) sums_of(i, f);
        part[2 * i * kTile + m] = make_float4(f[0], f[1], f[2], f[3]);
        part[(2 * i + 1) * kTile + m] = make_float4(f[4], f[5], f[6], f[7]);
      }
    cl.sync();
    if (warp < kMmaWarp)
      for (int i = first; i < n8; i += stride) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int cc = 0; cc < csize; cc += 4) {        // four CTAs' loads in flight, added in rank order
          float4 v[4][2];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[c][0] = v[c][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (cc + c < csize) {
              const float4* p = cl.map_shared_rank(part, cc + c) + 2 * i * kTile + m;
              v[c][0] = p[0];
              v[c][1] = p[kTile];
            }
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f[0] += v[c][0].x; f[1] += v[c][0].y; f[2] += v[c][0].z; f[3] += v[c][0].w;
            f[4] += v[c][1].x; f[5] += v[c][1].y; f[6] += v[c][1].z; f[7] += v[c][1].w;
          }
        }
        write(i, f);
      }
    cl.barrier_arrive();                               // partial sums stay until every CTA has read them
  }
  if (DIR == 0 && a.u && rank == 0 && mine && half == 0)
    for (int c = rp; c < R; c += 4) *reinterpret_cast<float4*>(a.u + grow * R + c) = make_float4(0.f, 0.f, 0.f, 0.f);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  free_tmem();
  if (csize > 1) cl.barrier_wait();
}

// ---------------------------------------------------------------------------
// second product
// ---------------------------------------------------------------------------
// kDirect (R <= 32): a lane loads its row of the operand itself; else the rows come
// through shared memory, as a lane's 16 bytes are half a sector of a row of its own
// (us, direct and through shared memory: 8191 rows at rank 64 30.8 and 28.3, at rank 16
// 24.6 and 25.4; the gradient of 16380 rows at rank 32 79.6 and 82.2).
template <int RB, bool kDirect>
struct Expand {
  static constexpr uint32_t kStageBytes = kXBytes + RB * 8192;
  static constexpr int kPerSM = RB == 1 ? 2 : 1;
  static constexpr int kStages = kDirect || RB == 2 ? 4 : 3;   // 96 / 72 / 128 KB
  static constexpr uint32_t kRowBytes = kDirect ? 0 : RB * 256;   // a row of the operand in fp32, behind the ring: 32 / 64 KB
  // TMEM: outputs of 64 columns, then the operand's terms, two BF16 a column
  static constexpr int kOuts = RB == 1 ? 2 : 4;
  static constexpr uint32_t kOperand = 64 * kOuts, kTerm = 32 * RB;
  static constexpr uint32_t kTmemCols = RB == 1 ? 256 : 512;
  static constexpr int kDrainWarps = 8;                // two groups, taking steps in turn
  static constexpr int kThreads = 32 * (kDrainWarps + 1 + kLoadWarps);
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kTile * kRowBytes;
};

template <int DIR, int RB, bool kDirect>
__global__ void __launch_bounds__(Expand<RB, kDirect>::kThreads, Expand<RB, kDirect>::kPerSM) lora_expand_kernel(const TileArgs a) {
  using L = Expand<RB, kDirect>;
  constexpr int kStages = L::kStages, kDrainWarps = L::kDrainWarps, kOuts = L::kOuts;
  constexpr uint32_t kTmemCols = L::kTmemCols;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], used[kStages], operand, out_full[kOuts], out_free[kOuts], last;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  __shared__ Unit unit_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int index = (int)(gridDim.x - 1 - blockIdx.x), part = index % a.parts;
  if (warp == 0) {
    const Unit u = find_unit(a.offsets, a.G, a.T, kTile, a.out != a.base, index / a.parts);
    if (lane == 0) unit_s = u;
  }
  if (warp == kDrainWarps) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) {
        mbar_init(&full[s], kLoaders);
        mbar_init(&used[s], kDrainWarps / 2);
      }
      mbar_init(&operand, 32 * kDrainWarps);
      mbar_init(&last, 1);
      for (int i = 0; i < kOuts; ++i) {
        mbar_init(&out_full[i], 1);
        mbar_init(&out_free[i], kDrainWarps / 2);
      }
      failed = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // dA's and dB's CTAs may come as SMs free up; TMEM is this CTA's by now
  if (DIR == 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  auto free_tmem = [&]() {
    // the launch does not end before the shrink has, whatever its CTAs had to do
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == kDrainWarps)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  };
  const Unit un = unit_s;
  const Guard guard{&failed, a.limit};
  const int K2 = a.K2, R = a.R, g = un.g;
  const int c_all = (K2 + kStep - 1) / kStep, c_per = (c_all + a.parts - 1) / a.parts;
  const int cb = min(c_all, part * c_per), nc = min(c_all, cb + c_per) - cb;
  if (un.rows == 0 || nc == 0) return free_tmem();
  int tok[8];
  const int q = warp & 3, half = warp >> 2;            // drain warps: TMEM lane quarter and group
  if (warp > kDrainWarps) {
    tile_tokens(tok, a, un, tid - 32 * (kDrainWarps + 1));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {                      // the rows this lane writes: q*32 + lane/8 + 4j
      const int r = q * 32 + (lane >> 3) + 4 * j;
      tok[j] = r < un.rows ? token_of(a.token_of_row, un.row0 + r, a.T) : -1;
    }
  }
  const int rk = g < a.G ? rank_of(a.rank, g, R) : 0;
  if (rk == 0) {                                       // no adapter: out = base
    if (a.out == a.base) return free_tmem();
    const int v8 = (min(K2, (cb + nc) * kStep) - cb * kStep) / 8;
    for (int r = warp; r < un.rows; r += 8 * (L::kThreads / 32)) {
      int t[8];                                        // eight rows in flight: one at a time took 10 us a tile
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = r + j * (L::kThreads / 32);
        t[j] = row < un.rows ? token_of(a.token_of_row, un.row0 + row, a.T) : -1;
      }
      for (int c = lane; c < v8; c += 32) {
        const size_t at = (size_t)cb * kStep + 8 * c;
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = make_uint4(0, 0, 0, 0);
          if (a.base && t[j] >= 0) v[j] = *reinterpret_cast<const uint4*>(a.base + (size_t)t[j] * K2 + at);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (t[j] >= 0) *reinterpret_cast<uint4*>(a.out + (size_t)t[j] * K2 + at) = v[j];
      }
    }
    return free_tmem();
  }
  const int rp = (rk + 15) & ~15;                      // the MMAs' K
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem), full_a = smem_u32(full), used_a = smem_u32(used);

  if (warp > kDrainWarps) {
    // ------------------------------------------------------------------ load
    const int l = tid - 32 * (kDrainWarps + 1);
    const uint32_t xo = place(l >> 3, l & 7, 0);
    Rows rows(a.base, a.w2, tok, K2, l, cb);
    Weights<RB, DIR == 1> w(a.w2, g, K2, R, rk, rp, l, cb);
    Ring<kStages> at;
    auto step = [&]() {
      const uint32_t st = ring + at.slot * L::kStageBytes;
      rows.load(st + xo, 1);
      w.load(st + kXBytes, xo, 1);
      cp_arrive(full_a + 8 * at.slot);
      at.next();
    };
    // base and weights do not depend on the shrink, and do not wait for it
    const int ahead = min(nc, kStages);
    for (int s = 0; s < ahead && !a.drop; ++s) step();
    for (int s = ahead; s < nc && !a.drop; ++s) {
      wait_bar(used_a + 8 * at.slot, at.parity ^ 1u, guard);
      step();
    }
    cp_wait_all();
  } else if (warp == kDrainWarps) {
    // ------------------------------------------------------------------ MMAs
    const uint32_t go = elect_one(), id = idesc(kStep, 0, DIR);
    Ring<kStages> at;
    const uint64_t dw0 = DIR ? desc_mn(ring + kXBytes, 8192) : smem_desc(ring + kXBytes);
    const uint32_t of = smem_u32(out_full), fr = smem_u32(out_free);
    wait_bar(smem_u32(&operand), 0, guard);
    tc_fence_after();
#pragma unroll 1
    for (int o = 0; o < nc; ++o) {
      const int buf = o % kOuts;
      wait_bar(full_a + 8 * at.slot, at.parity, guard);
      if (o >= kOuts) {
        wait_bar(fr + 8 * buf, (uint32_t)(o / kOuts - 1) & 1u, guard);
        tc_fence_after();
      }
      fence_async();
      const uint64_t dw = dw0 + at.slot * (L::kStageBytes >> 4);
      const uint32_t d = tmem + 64 * (uint32_t)buf;
#pragma unroll 1
      for (int term = 2; term >= 0; --term)            // the small terms first: their sums lose nothing
#pragma unroll 1
        for (int kk = 0; 16 * kk < rp; ++kk)
          mma_ts(d, tmem + L::kOperand + term * L::kTerm + 8 * kk,
                 dw + (DIR ? (2048 >> 4) * kk : (kk >> 2) * (8192 >> 4) + 2 * (kk & 3)), id, term != 2 || kk != 0, go);
      commit_at(of + 8 * buf, go);
      at.next();
    }
    finish_mmas(&last, go, a.limit);
  } else {
    // ------------------------------------------------------------------ operand
    // The first product's sums into TMEM in three BF16 terms, a row a lane, every other
    // eight columns.  They were written beside this launch's beginning: loads past L1.
    const int m = q * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    {
      const int c_end = rp / 8, c_in = min(rp, R) / 8; // zeros between them
      const uint8_t* staged = smem + kStages * L::kStageBytes + m * L::kRowBytes;
      if (!kDirect) {
        const uint32_t op = ring + kStages * L::kStageBytes;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = (tid >> 3) + 32 * j;
          const float* p = a.second + (size_t)(un.row0 + min(row, un.rows - 1)) * R;
#pragma unroll
          for (int e = 0; e < 2 * RB; ++e) {
            const int c = (tid & 7) + 8 * e;           // of four columns, 128-byte swizzled
            if (c < 2 * c_in) cp16(op + row * L::kRowBytes + 16u * (uint32_t)(c ^ (row & 7)), p + 4 * c);
          }
        }
        cp_wait_all();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * L::kDrainWarps) : "memory");
      }
      const float4* row = reinterpret_cast<const float4*>(a.second + (size_t)(un.row0 + min(m, un.rows - 1)) * R);
      float4 v[4 * RB][2];
#pragma unroll
      for (int e = 0; e < 4 * RB; ++e) {
        const int c = half + 2 * e;
        v[e][0] = v[e][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < c_in) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            v[e][h] = kDirect ? __ldcg(row + 2 * c + h) : *reinterpret_cast<const float4*>(staged + 16 * ((2 * c + h) ^ (m & 7)));
        }
      }
#pragma unroll
      for (int e = 0; e < 4 * RB; ++e) {
        const int c = half + 2 * e;
        if (c < c_end) {
          uint4 t[3];
          split8(v[e], t);
#pragma unroll
          for (int i = 0; i < 3; ++i)
            tmem_st4(tmem + ((uint32_t)(q * 32) << 16) + L::kOperand + i * L::kTerm + 4 * (uint32_t)c, t[i]);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&operand);
    }
    // ------------------------------------------------------------------ outputs
    // base (in the ring) plus product, one rounding.  The two groups of four
    // warps take alternate steps, so that one's latencies hide behind the other's
    const uint32_t ro = place(q * 32 + (lane >> 3), lane & 7, 0), mo = place(m, 0, 0);
    Ring<kStages> at;
    if (half) at.next();
    const uint32_t of = smem_u32(out_full);
    for (int o = half; o < nc; o += 2) {
      const int buf = o % kOuts;
      uint8_t* xt = smem + (size_t)at.slot * L::kStageBytes;
      wait_bar(of + 8 * buf, (uint32_t)(o / kOuts) & 1u, guard);
      wait_bar(full_a + 8 * at.slot, at.parity, guard);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t d[2][16];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + 64u * (uint32_t)buf + 32u * h, d[0], d[1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float b[8];
          uint4* p = reinterpret_cast<uint4*>(xt + (mo ^ (uint32_t)((4 * h + c) << 4)));
          unpack8(*p, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] += __uint_as_float(d[c >> 1][(c & 1) * 8 + e]);
          *p = make_uint4(pack2(b[0], b[1]), pack2(b[2], b[3]), pack2(b[4], b[5]), pack2(b[6], b[7]));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&out_free[buf]);
      const int col = (cb + o) * kStep + 8 * (lane & 7);
      if (col < K2) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (tok[j] >= 0)
            *reinterpret_cast<uint4*>(a.out + (size_t)(unsigned)tok[j] * (unsigned)K2 + col) =
                *reinterpret_cast<const uint4*>(xt + ((ro + 512u * j) ^ ((j & 1) << 6)));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&used[at.slot]);
      at.next();
      at.next();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  free_tmem();
}

// ---------------------------------------------------------------------------
// dA and dB
// ---------------------------------------------------------------------------
struct DwArgs {
  const uint16_t* src[2];                              // x [T, H], dy [T, N]
  const float* factor[2];                              // v, u: [T, R]
  uint16_t* out[2];                                    // da [G, R, H], db [G, N, R]
  const float* scale;
  const int32_t *rank, *offsets, *token_of_row;
  int M[2];                                            // H, N
  int T, G, R;
  long long limit;
  int drop;
};

// A step is 32 rows of 256 columns: 16 KB of x or dy and RB x 12 KB of the
// factor's three terms.  (With 128 columns the factor is read twice as often and
// there are twice as many CTAs to set up: 39 against 36 us for 60 groups of
// 273 rows, 2048 and 1408 columns, rank 32; 13.3 against 14.9 us for one group
// of 2047 rows.)
// kWide: R <= 32, the terms lie side by side as the columns of one product (3 R), so that
// an MMA reads the 128 columns of x or dy once for all of them; else a term has RB blocks
// of 64 columns (R <= 64 RB), and the second and third term's products share a sum.
// Either way the first term's sum is cut to fp32 once per MMA, not once per term.
template <int RB, bool kWide>
struct Dw {
  static constexpr int kRows = 32, kCols = 2 * kTile;
  static constexpr uint32_t kBlock = kRows * 128;      // 64 columns
  static constexpr uint32_t kSrcBytes = kRows * kCols * 2;
  static constexpr uint32_t kStageBytes = kSrcBytes + (kWide ? 2 : 3 * RB) * kBlock;
  static constexpr int kPerSM = RB == 1 ? 2 : 1;
  static constexpr int kStages = kWide ? 4 : RB == 1 ? 3 : 5;   // 96 / 84 / 200 KB
  static constexpr int kDepth = kWide ? 4 : 3;         // steps of the factor in registers
  static constexpr uint32_t kTileCols = kWide ? 96 : RB * 128;  // of TMEM, for 128 columns of x or dy
  static constexpr uint32_t kTmemCols = kWide ? 256 : 2 * kTileCols;
  static constexpr int kSmem = 1024 + kStages * kStageBytes;
};

// Four warps load x or dy and then drain, one issues the MMAs, four load and split the
// factor: in the first four it would hold up the copies of later steps.
constexpr int kDwThreads = 2 * kLoaders + 32;

template <int RB, bool kWide>
__global__ void __launch_bounds__(kDwThreads, Dw<RB, kWide>::kPerSM) lora_dw_kernel(const DwArgs a) {
  using D = Dw<RB, kWide>;
  constexpr int kStages = D::kStages, kRows = D::kRows;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], used[kStages], sums, last;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), csize = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // dB of every adapter first: it reads nothing of the launches in front and runs
  // beside them; dA waits
  const int unit = (int)(blockIdx.x / csize), unitsB = (a.M[1] + D::kCols - 1) / D::kCols * a.G;
  const int which = unit < unitsB, M = a.M[which], tiles = (M + D::kCols - 1) / D::kCols;
  const int index = which ? unit : unit - unitsB, g = index / tiles, m0 = (index - g * tiles) * D::kCols;
  const int R = a.R, rk = rank_of(a.rank, g, R);
  const int r0 = min(max(a.offsets[g], 0), a.T), r1 = min(max(a.offsets[g + 1], 0), a.T);
  uint16_t* out = a.out[which];

  // eight rank columns from c0 on of column m0 + tid (TMEM lane) + 128 t
  auto store = [&](int t, int c0, const float (&v)[8]) {
    const int m = m0 + t * kTile + tid;
    if (tid >= kTile || m >= M || c0 >= R) return;
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
  for (int c = rp / 8 + rank; c < R / 8; c += csize) {
    store(0, 8 * c, zero8);
    store(1, 8 * c, zero8);
  }
  // the launch does not end before the one in front has, whatever its CTAs had to do
  auto wait_last = [&]() {
    if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (rp == 0) return wait_last();                     // the whole cluster leaves

  const int s_all = (r1 - r0 + kRows - 1) / kRows, s_per = (s_all + csize - 1) / csize;
  const int sb = min(s_all, rank * s_per), ns = min(s_all, sb + s_per) - sb;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem), full_a = smem_u32(full), used_a = smem_u32(used);
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 2 * kLoaders);               // copies, and the factor's stores
      mbar_init(&used[s], 1);
    }
    mbar_init(&sums, 1);
    mbar_init(&last, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kLoadWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(D::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Guard guard{&failed, a.limit};

  if (warp == kLoadWarps) {
    // ------------------------------------------------------------------ MMAs
    {
      const uint32_t go = elect_one();
      const uint32_t id = idesc(kWide ? 3 * rp : rp, 1, 1);
      const uint64_t dx0 = desc_mn(ring, D::kBlock), dw0 = desc_mn(ring + D::kSrcBytes, D::kBlock);
      Ring<kStages> at;
#pragma unroll 1
      for (int s = 0; s < ns; ++s) {
        wait_bar(full_a + 8 * at.slot, at.parity, guard);
        fence_async();
        const uint32_t off = at.slot * (D::kStageBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          const uint64_t dw = dw0 + off + kk * (2048 >> 4);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint64_t da = dx0 + off + kk * (2048 >> 4) + n * (2 * D::kBlock >> 4);
#pragma unroll
            for (int i = kWide ? 0 : 2; i >= 0; --i)
              mma_ss(tmem + n * D::kTileCols + (i ? RB * 64 : 0), da, dw + i * (RB * D::kBlock >> 4), id, i == 1 || (s | kk) != 0, go);
          }
        }
        commit_at(used_a + 8 * at.slot, go);
        at.next();
      }
      commit_at(smem_u32(&sums), go);
      finish_mmas(&last, go, a.limit);
    }
    __syncwarp();
  } else if (warp > kLoadWarps) {
    // ------------------------------------------------------------------ factor
    // Pieces of eight columns of a row, kDepth steps ahead in fp32 (a step waits a load's
    // latency / kDepth) and past L1, as the shrink may run beside this launch's beginning.
    constexpr int kPieces = kWide ? 1 : 2 * RB, kDepth = D::kDepth;
    const int l = tid - 32 * (kLoadWarps + 1);
    const int n8 = min(rp, R) / 8;                     // chunks in memory; zeros behind them up to rp / 8
    int row[kPieces], chunk[kPieces];
    uint32_t at3[kPieces][3];                          // the terms' places; 0: not a piece
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int sh = !kWide ? 3 : rp > 16 ? 2 : 1;     // kWide: 2 or 4 chunks a row
      row[i] = (l >> sh) + 16 * (i & 1);
      chunk[i] = (l & ((1 << sh) - 1)) + 8 * (i >> 1);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        at3[i][q] = row[i] < kRows && chunk[i] < rp / 8
                        ? D::kSrcBytes + place(row[i], kWide ? q * (rp / 8) + chunk[i] : 8 * RB * q + chunk[i], D::kBlock)
                        : 0u;
    }
    const float* factor = a.factor[which];
    float4 held[kDepth][kPieces][2];
    auto load = [&](float4 (&h)[kPieces][2], int s) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = r0 + (sb + s) * kRows + row[i];
        h[i][0] = h[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < ns && r < r1 && row[i] < kRows && chunk[i] < n8) {
          const float4* p = reinterpret_cast<const float4*>(factor + (size_t)r * R + 8 * chunk[i]);
          h[i][0] = __ldcg(p);
          h[i][1] = __ldcg(p + 1);
        }
      }
    };
    if (!which) asm volatile("griddepcontrol.wait;" ::: "memory");   // v is the shrink's
#pragma unroll
    for (int e = 0; e < kDepth; ++e) load(held[e], e);
    Ring<kStages> at;
    for (int s0 = 0; s0 < ns && !a.drop; s0 += kDepth) {
#pragma unroll
      for (int e = 0; e < kDepth; ++e) {
        const int s = s0 + e;
        if (s >= ns) break;
        if (s >= kStages) wait_bar(used_a + 8 * at.slot, at.parity ^ 1u, guard);
        const uint32_t st = ring + at.slot * D::kStageBytes;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          if (at3[i][0]) {
            uint4 t[3];
            split8(held[e][i], t);
#pragma unroll
            for (int q = 0; q < 3; ++q) st16(st + at3[i][q], t[q]);
          }
        }
        arrive_at(full_a + 8 * at.slot);               // (the MMA warp's fence covers the stores)
        load(held[e], s + kDepth);
        at.next();
      }
    }
  } else {
    // ------------------------------------------------------------------ loaders
    // 32 rows x 256 columns of src per step: this thread's chunk (its lane) of rows
    // warp + 4j
    const int col = m0 + 8 * lane;
    uint32_t xo[2];
    xo[0] = place(warp, lane, D::kBlock);              // + 1024 every eight rows
    xo[1] = place(warp + 4, lane, D::kBlock);
    const uint16_t* src = a.src[which];
    const int first = r0 + sb * kRows;
    const int xbytes = col < M ? 16 : 0;
    const uint16_t* xsrc = xbytes ? src + col : src;
    // tokens: lane l holds row l of each of four steps, loaded four steps ahead
    int cur[4], nxt[4];
    auto load_tok = [&](int (&t)[4], int s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = first + (s + i) * kRows + lane;
        t[i] = s + i < ns && row < r1 ? (a.token_of_row ? __ldg(a.token_of_row + row) : row) : -1;
      }
    };
    load_tok(cur, 0);
    Ring<kStages> at;
    for (int s0 = 0; s0 < ns && !a.drop; s0 += 4) {
      load_tok(nxt, s0 + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = s0 + e;
        if (s >= ns) break;
        if (s >= kStages) wait_bar(used_a + 8 * at.slot, at.parity ^ 1u, guard);
        const uint32_t st = ring + at.slot * D::kStageBytes;
#pragma unroll
        for (int j = 0; j < kRows / 4; ++j) {
          const int t = __shfl_sync(kFull, cur[e], warp + 4 * j);
          const bool in = (unsigned)t < (unsigned)a.T;
          cp16(st + xo[j & 1] + 1024u * (j >> 1), in ? xsrc + (size_t)(unsigned)t * (unsigned)M : src, in ? xbytes : 0);
        }
        cp_arrive(full_a + 8 * at.slot);
        at.next();
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) cur[e] = nxt[e];
    }
    cp_wait_all();
    wait_bar(smem_u32(&sums), 0, guard);             // every MMA has read the ring
    tc_fence_after();
  }
  __syncthreads();                                     // the ring is free: partial sums take its place
  float4* part = reinterpret_cast<float4*>(smem);      // [2][rp / 4][kTile][4]
  const float scale = which && a.scale ? a.scale[g] : 1.0f;
  const int n8 = rp / 8;
  if (warp < kLoadWarps) {
    for (int c = 0; c < 2 * n8; ++c) {                 // tile c / n8, rank columns 8 (c % n8) on
      const int t = c >= n8, c8 = 8 * (c - t * n8);
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (ns > 0) {
        const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(t * D::kTileCols + c8);
        constexpr int kSums = kWide ? 3 : 2;
        uint32_t w[kSums][8];
#pragma unroll
        for (int q = 0; q < kSums; ++q) tmem_ld8(at + q * (kWide ? rp : RB * 64), w[q]);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = __uint_as_float(w[kSums - 1][e]);     // the small sums first
#pragma unroll
          for (int q = kSums - 2; q >= 0; --q) v[e] += __uint_as_float(w[q][e]);
        }
      }
      if (csize > 1) {
        part[(2 * c) * kTile + tid] = make_float4(v[0], v[1], v[2], v[3]);
        part[(2 * c + 1) * kTile + tid] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c8 + e < rk ? v[e] * scale : 0.0f;
        store(t, c8, v);
      }
    }
  }
  if (csize > 1) {
    cl.sync();
    if (warp < kLoadWarps) {
      for (int c = rank; c < 2 * n8; c += csize) {
        const int t = c >= n8, c8 = 8 * (c - t * n8);
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int pc = 0; pc < csize; pc += 4) {        // four CTAs' loads in flight, added in rank order
          float4 w[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i][0] = w[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (pc + i < csize) {
              const float4* p = cl.map_shared_rank(part, pc + i) + 2 * c * kTile + tid;
              w[i][0] = p[0];
              w[i][1] = p[kTile];
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[0] += w[i][0].x; v[1] += w[i][0].y; v[2] += w[i][0].z; v[3] += w[i][0].w;
            v[4] += w[i][1].x; v[5] += w[i][1].y; v[6] += w[i][1].z; v[7] += w[i][1].w;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c8 + e < rk ? v[e] * scale : 0.0f;
        store(t, c8, v);
      }
    }
    cl.sync();                                         // partial sums stay until every CTA has read them
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kLoadWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(D::kTmemCols) : "memory");
  }
  wait_last();
}
template <class K, class A>
zmoe_status launch(K* kernel, dim3 grid, int threads, int csize, bool dependent, int smem, cudaStream_t stream,
                   const A& args, const char* what) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, kernel, args));
  return launch_status(what);
}

// How many CTAs share a unit of `steps` steps: the count with the least rounds x
// (steps of a CTA + fixed), where a round fills the `places` of the SMs and
// `fixed` is what a CTA spends around its steps, in steps.
int share(long long units, int steps, int places, int fixed, int fixed_shared, int most, bool powers) {
  int best = 1;
  long long least = -1;
  for (int c = 1; c <= most && c <= steps; c = powers ? 2 * c : c + 1) {
    const long long rounds = (units * c + places - 1) / places;
    const long long cost = rounds * ((steps + c - 1) / c + (c > 1 ? fixed_shared : fixed));
    if (least < 0 || cost < least) {
      least = cost;
      best = c;
    }
  }
  return best;
}

template <int DIR, int RB, bool kDirect>
zmoe_status launch_tiles(TileArgs a, cudaStream_t stream) {
  const long long units = a.T / kTile + (a.T < a.G + 2 ? a.T : a.G + 2);       // at most
  const int tiles = (a.T + kTile - 1) / kTile + (a.T < a.G ? a.T : a.G) / 2;   // about
  using S = Shrink<RB>;
  using E = Expand<RB, kDirect>;
  zmoe_status st = allow_smem<lora_shrink_kernel<DIR, RB>>();
  if (st == ZMOE_OK) st = allow_smem<lora_expand_kernel<DIR, RB, kDirect>>();
  if (st != ZMOE_OK) return st;
  const int c = share(tiles, (a.K1 + kStep - 1) / kStep, kNumSMs * S::kPerSM, 2, 8, 8, true);
  const int steps2 = (a.K2 + kStep - 1) / kStep;
  if (a.weights >= kNumSMs) {
    // dB runs beside dx and fills the other half of the SMs: about one CTA an SM, of four
    // steps at least (us with the forward's rule and with this one: 16380 rows of 60
    // adapters, 3 parts and 1, 82.8 and 79.5; 2047 rows of one, whose dB is 32 CTAs, 16
    // parts and 9, 29.2 and 31.5)
    a.parts = (kNumSMs + tiles / 2) / tiles;
    a.parts = a.parts > steps2 / 4 ? steps2 / 4 : a.parts;
    a.parts = a.parts < 1 ? 1 : a.parts;
  } else {
    a.parts = share(tiles, steps2, kNumSMs * E::kPerSM, 5, 5, 64, false);
  }
  ZMOE_CHECK_ARG(units * c < (1LL << 31) && units * a.parts < (1LL << 31), "lora: T=%d rows are too many for one launch",
                 a.T);
  st = launch(lora_shrink_kernel<DIR, RB>, dim3((unsigned)(units * c)), S::kThreads, c, false, S::kSmem, stream, a,
              "lora_shrink_kernel");
  if (st != ZMOE_OK || !a.out) return st;
  return launch(lora_expand_kernel<DIR, RB, kDirect>, dim3((unsigned)(units * a.parts)), E::kThreads, 1, true, E::kSmem, stream, a,
                "lora_expand_kernel");
}

template <int DIR>
zmoe_status launch_tiles(const TileArgs& a, cudaStream_t stream) {
  return a.R <= 32   ? launch_tiles<DIR, 1, true>(a, stream)
         : a.R <= 64 ? launch_tiles<DIR, 1, false>(a, stream)
                     : launch_tiles<DIR, 2, false>(a, stream);
}

template <int RB, bool kWide>
zmoe_status launch_dw(const DwArgs& a, cudaStream_t stream) {
  using D = Dw<RB, kWide>;
  zmoe_status st = allow_smem<lora_dw_kernel<RB, kWide>>();
  if (st != ZMOE_OK) return st;
  const int tiles = (a.M[0] + D::kCols - 1) / D::kCols + (a.M[1] + D::kCols - 1) / D::kCols;
  const int steps = (a.T + D::kRows - 1) / D::kRows;
  const long long units = (long long)tiles * a.G;
  const int most = steps / a.G / 5;
  // One adapter: as many CTAs as there are SMs.  Several have uneven rows: up to 4 CTAs
  // a tile while they are not far too many, so that the longest does not end alone.
  // Five steps each at least.
  // (us: 2047 rows of one, 30 tiles x 4 CTAs 29.2, x 8 29.8; 8192 rows of 4, 64 tiles x
  // 2 52.9, x 4 46.6; 65536 rows of 16, 256 tiles x 2 260, x 4 244, x 8 265; 32768 rows
  // of 60 experts, 840 tiles x 1 124, x 2 148.  All with rows in every group: the host
  // does not know the rows, so a bank of G adapters of which one is used is shared like G.)
  int csize = 1;
  while (csize < 8 && csize * 2 <= most && units * csize * 2 <= (a.G > 1 && csize < 4 ? 8 * kNumSMs : kNumSMs)) csize *= 2;
  return launch(lora_dw_kernel<RB, kWide>, dim3((unsigned)(units * csize)), kDwThreads, csize, true,
                D::kSmem, stream, a, "lora_dw_kernel");
}

}  // namespace

zmoe_status launch_tiles(const zmoe_lora_args* p, cudaStream_t stream) {
  const TileArgs a{p->x, p->a, p->b, p->base, p->scale, p->rank, p->offsets, p->token_of_row, p->T, p->H, p->N, p->G,
                   p->R, p->out, p->u, p->scratch, 0, 1, tc::wait_limit(), tc::drop_loads()};
  return launch_tiles<0>(a, stream);
}

zmoe_status launch_grad_tiles(const zmoe_lora_grad_args* p, cudaStream_t stream) {
  const TileArgs a{p->dy, p->b, p->a, p->base, p->scale, p->rank, p->offsets, p->token_of_row, p->T, p->N, p->H, p->G,
                   p->R, p->dx, nullptr, p->scratch, p->da ? (long long)p->G * ((p->N + 2 * kTile - 1) / (2 * kTile)) : 0, 1, tc::wait_limit(), tc::drop_loads()};
  zmoe_status st = launch_tiles<1>(a, stream);
  if (st != ZMOE_OK || !p->da) return st;
  const DwArgs d{{p->x, p->dy}, {p->scratch, p->u}, {p->da, p->db}, p->scale, p->rank, p->offsets, p->token_of_row,
                 {p->H, p->N}, p->T, p->G, p->R, tc::wait_limit(), tc::drop_loads()};
  return p->R <= 32 ? launch_dw<1, true>(d, stream) : p->R <= 64 ? launch_dw<1, false>(d, stream) : launch_dw<2, false>(d, stream);
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
