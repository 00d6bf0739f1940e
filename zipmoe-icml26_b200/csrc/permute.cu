// Permute (K3): per-expert counts, capacity drops, row assignment and the
// activation gather.
//
// Reference: ExpertExecutor.dispatch_local counts tokens per expert
// (experts/expert_executor.py:45-49) and ExpertDispatcher::GPUFetchFunc
// gathers them with a boolean mask, tokens ascending
// (csrc/dispatcher/expert_dispatcher.cpp:326-330).  The Switch capacity mask
// is the cumsum over the sequence axis of the transformers<4.47 Top1 router.
//
// Without a capacity the order is a stable counting sort of the (token, slot)
// pairs by expert.  Each warp of a cluster of CTAs takes a run of tokens, and
// counts its experts in its own shared-memory row (lanes with the same expert
// find each other by votes, so a step of 32 pairs is one add per expert
// present); prefixes over warps, CTAs (through distributed shared memory) and
// experts turn the counts into first rows, and a second walk over the same
// pairs hands the rows out in order.  No atomics: the result does not depend
// on timing.  The activation rows are then copied token by token, so that x is
// read once and each row is written once.
//   * up to kFusedPairs pairs: one launch; every CTA sorts all pairs for
//     itself and copies its own share of the rows, so that nothing waits on
//     another CTA;
//   * more: one cluster sorts, and the copy follows as a dependent launch that
//     loads x while the sort finishes;
//   * from kWidePairs on: CTAs of an ordinary launch count their shares, one CTA
//     turns the counts into first rows, and the CTAs place their pairs.
//
// With a capacity (Switch) drops depend on the rank within a sequence, and
// three small launches do it: (1) one CTA per expert ranks its tokens in token
// order with a block scan, drops those past the capacity of their sequence and
// writes the count; (2) one CTA per expert turns counts into offsets and writes
// row_of / token_of_row in the same order; (3) the copy.  They also take what
// the sort's shared memory and steps do not hold (more than kSortE experts,
// more than 32 slots).
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace zmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxT = 0x7fffffff - kThreads;           // a step behind the last token still is an int

// Exclusive block scan of v (0/1 flags); returns the prefix, *total gets the sum.
__device__ __forceinline__ int block_exclusive_scan(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (threadIdx.x < 32) {
    int s = threadIdx.x < kThreads / 32 ? warp_sums[threadIdx.x] : 0;
    int si = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, si, d);
      if ((int)threadIdx.x >= d) si += o;
    }
    if (threadIdx.x < kThreads / 32) warp_sums[threadIdx.x] = si - s;   // exclusive
    if (threadIdx.x == kThreads / 32 - 1) warp_sums[kThreads / 32] = si;
  }
  __syncthreads();
  const int r = warp_sums[warp] + incl - v;
  *total = warp_sums[kThreads / 32];
  __syncthreads();
  return r;
}

__device__ __forceinline__ int slot_of(const int32_t* idx, int t, int k, int e) {
  for (int j = 0; j < k; ++j)
    if (idx[(size_t)t * k + j] == e) return j;
  return -1;
}

__global__ void __launch_bounds__(kThreads)
count_kernel(int32_t* __restrict__ topk_idx, int T, int k, int capacity, int seq_len,
             int32_t* __restrict__ counts) {
  __shared__ int warp_sums[kThreads / 32 + 1];
  const int e = blockIdx.x;
  const int row_len = capacity > 0 ? seq_len : T;
  int kept = 0;
  for (int r0 = 0; r0 < T; r0 += row_len) {
    const int r1 = min(T, r0 + row_len);
    int running = 0;
    for (int t0 = r0; t0 < r1; t0 += kThreads) {
      const int t = t0 + threadIdx.x;
      const int j = t < r1 ? slot_of(topk_idx, t, k, e) : -1;
      int total;
      const int rank = running + block_exclusive_scan(j >= 0 ? 1 : 0, warp_sums, &total);
      const bool drop = j >= 0 && capacity > 0 && rank >= capacity;
      if (drop) topk_idx[(size_t)t * k + j] = -1;
      kept += __syncthreads_count(j >= 0 && !drop);
      running += total;
    }
  }
  if (threadIdx.x == 0) counts[e] = kept;
}

__global__ void __launch_bounds__(kThreads)
scatter_kernel(const int32_t* __restrict__ topk_idx, int T, int k, int E,
               const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
               int32_t* __restrict__ row_of, int32_t* __restrict__ token_of_row) {
  __shared__ int warp_sums[kThreads / 32 + 1];
  __shared__ int base_s;
  const int e = blockIdx.x;
  if (threadIdx.x == 0) {
    int s = 0;
    for (int q = 0; q < e; ++q) s += counts[q];
    base_s = s;
    if (e == E - 1) {
      int acc = 0;
      for (int q = 0; q < E; ++q) { offsets[q] = acc; acc += counts[q]; }
      offsets[E] = acc;
    }
  }
  __syncthreads();
  const int base = base_s;
  int running = 0;
  for (int t0 = 0; t0 < T; t0 += kThreads) {
    const int t = t0 + threadIdx.x;
    const int j = t < T ? slot_of(topk_idx, t, k, e) : -1;
    int total;
    const int rank = running + block_exclusive_scan(j >= 0 ? 1 : 0, warp_sums, &total);
    if (j >= 0) {
      const int row = base + rank;
      row_of[(size_t)t * k + j] = row;
      token_of_row[row] = t;
    }
    running += total;
  }
}

// ---------------------------------------------------------------------------
// counting sort
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortE = 1024;          // experts: one per thread in the scan, 128 KB of warp counts
constexpr int kSortCluster = 16;      // the steps are bound by instruction issue: 98 thousand
                                      // pairs took 19 us on 8 SMs, 12 on 16
constexpr int kFusedPairs = 1024;     // pairs every CTA of the fused launch sorts for itself
                                      // (64 experts, rows of 2048, us, fused against two launches: 64 pairs of 4 a
                                      // token 4.8 and 6.1, of 8 a token 4.6 and 6.1; 1024 pairs 5.6 and 6.7; 2048 pairs
                                      // 7.7 and 7.7, at rows of 1024 7.2 and 6.9, of 4096 10.0 and 9.2)
constexpr int kWidePairs = 131072;    // pairs from which the sort takes three launches of kWideCtas CTAs instead of
constexpr int kWideCtas = 64;         // one cluster (with the copy of rows of 2048, us: 65536 pairs 73.8 and 70.8, 98 thousand
                                      // 87.3 and 87.2, 393 thousand 313 and 357; 128 CTAs 312).  All launches fit the SMs together
constexpr int kHold = 16;             // steps of a warp whose pairs stay in registers between the two walks
constexpr unsigned kFull = 0xffffffffu;

struct SortArgs {
  const int32_t* idx;                 // [T, k]
  int T, k, E;
  int rest;                           // 1: ids outside [0, E - 1) belong to the last group; 0: they have no row
  int32_t* counts;                    // [E] or nullptr
  int32_t* offsets;                   // [E + 1]; with rest the first E entries
  int32_t* row_of;                    // [T, k] or nullptr
  int32_t* token_of_row;              // [T * k] or nullptr: the copy of the rows writes it
  int wide;                           // sort in three launches: steps per warp; else 0
};

// The wide sort's CTAs: all but the last keep their counts, and then their first
// rows, in row_of at their own first token, where they are the only ones to write
// in the end; the last one keeps its counts in the output `counts`.
__device__ __forceinline__ int32_t* wide_counts(const SortArgs& a, int cta, int ctas) {
  return cta == ctas - 1 ? a.counts : a.row_of + (size_t)cta * kSortWarps * a.wide * (32 / a.k) * a.k;
}

// Sorts the pairs of tokens [0, T) by expert over the CTAs of a cluster (rank
// of csize).  smem: hist [kSortWarps][E], tot [E], base [E], warp_sums.
// write: this CTA writes the outputs in global memory.  rows_s (or nullptr)
// receives every pair's row in shared memory.
// kWide: the CTA is one of an ordinary launch: 1 writes its counts, 2 reads its first rows.
template <int kWide>
__device__ void sort_pairs(const SortArgs& a, int rank, int csize, int* smem, bool write, int32_t* rows_s) {
  int* hist = smem;
  int* tot = hist + kSortWarps * a.E;
  int* base = tot + a.E;
  int* warp_sums = base + a.E;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = a.k, E = a.E;
  const int tp = 32 / k;                               // whole tokens per step of a warp
  const int nw = kSortWarps * csize;
  const int steps_all = (a.T + tp - 1) / tp;
  const int per = kWide ? a.wide : (steps_all + nw - 1) / nw;   // steps per warp
  const int s0 = min(steps_all, (rank * kSortWarps + warp) * per), s1 = min(steps_all, s0 + per);
  const int jl = lane % k, tl = lane / k;              // slot and token of this lane in a step
  const bool used = tl < tp;
  const unsigned earlier = ((1u << lane) - 1u) & ~((1u << (lane - jl)) - 1u);   // same token, lower slots
  int* my = hist + warp * E;

  for (int e = lane; e < E; e += 32) my[e] = 0;
  __syncwarp();

  // A step's pair of this lane as seen by the warp: expert, earlier lanes with
  // the same expert << 10, lanes with it << 16; -1: no row, -2: no pair.
  auto load = [&](int s) -> int {
    if (!used || s >= s1) return -2;
    const int t = s * tp + tl;
    if (t >= a.T) return -2;
    const int e = __ldg(a.idx + (size_t)t * k + jl);
    if (a.rest) return (unsigned)e < (unsigned)(E - 1) ? e : E - 1;
    return (unsigned)e < (unsigned)E ? e : -1;
  };
  auto pack = [&](int e) -> int {
    // lanes with the same expert: one vote per bit of it (a match.any instead
    // took 0.3 us less for 256 pairs and 2 us more for 8192 on one SM)
    unsigned m = __ballot_sync(kFull, e >= 0);
#pragma unroll
    for (int b = 0; b < 10; ++b) {
      if (E <= 1 << b) break;
      const unsigned v = __ballot_sync(kFull, e >> b & 1);
      m &= e >> b & 1 ? v : ~v;
    }
    if (e >= 0 && (m & earlier)) e = -1;               // an expert named twice by a token counts once
    m &= __ballot_sync(kFull, e >= 0);
    return e < 0 ? e : e | __popc(m & ((1u << lane) - 1u)) << 10 | __popc(m) << 16;
  };
  auto count = [&](int v) {                            // the first lane of an expert adds for all
    if (v >= 0 && !(v >> 10 & 63)) my[v & 1023] += v >> 16;
    __syncwarp();
  };

  int held[kHold];
  const bool hold = per <= kHold;
  if (hold) {
#pragma unroll
    for (int b = 0; b < kHold; ++b) held[b] = load(s0 + b);
#pragma unroll
    for (int b = 0; b < kHold; ++b) {
      if (b >= per) break;
      held[b] = pack(held[b]);
      count(held[b]);
    }
  } else {
    for (int s = s0; s < s1; s += kHold) {
#pragma unroll
      for (int b = 0; b < kHold; ++b) held[b] = load(s + b);
#pragma unroll
      for (int b = 0; b < kHold; ++b) count(pack(held[b]));
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kSortThreads) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = hist[w * E + e];
      hist[w * E + e] = run;
      run += n;
    }
    if (kWide == 1) wide_counts(a, rank, csize)[e] = run;
    else tot[e] = run;
  }
  if (kWide == 1) return;
  const int e1 = threadIdx.x;
  if (kWide == 2) {
    asm volatile("griddepcontrol.wait;" ::: "memory"); // the counts have become first rows
    if (e1 < E) {
      const bool last = rank == csize - 1;             // its rows end an expert's
      const int32_t* p = last ? a.offsets + e1 + 1 : wide_counts(a, rank, csize) + e1;
      int n;
      asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(n) : "l"(p) : "memory");
      base[e1] = last ? n - tot[e1] : n;
    }
  } else {
    if (csize > 1) cg::this_cluster().sync();
    else __syncthreads();
    int all = 0, before = 0;
    if (e1 < E) {
      if (csize > 1) {
        int n[kSortCluster];
#pragma unroll
        for (int c = 0; c < kSortCluster; ++c) n[c] = c < csize ? *cg::this_cluster().map_shared_rank(tot + e1, c) : 0;
#pragma unroll
        for (int c = 0; c < kSortCluster; ++c) {
          if (c < rank) before += n[c];
          all += n[c];
        }
      } else {
        all = tot[e1];
      }
    }
    int incl = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(kFull, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int v = warp_sums[lane], si = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(kFull, si, d);
        if (lane >= d) si += o;
      }
      warp_sums[lane] = si - v;
    }
    __syncthreads();
    if (e1 < E) {
      const int first = warp_sums[warp] + incl - all;
      base[e1] = first + before;
      if (write && rank == 0) {
        if (a.counts) a.counts[e1] = all;
        a.offsets[e1] = first;
        if (e1 == E - 1 && !a.rest) a.offsets[E] = first + all;
      }
    }
  }
  __syncthreads();

  auto place = [&](int s, int v) {
    const int row = v >= 0 ? base[v & 1023] + my[v & 1023] + (v >> 10 & 63) : -1;
    __syncwarp();
    count(v);
    if (v >= -1) {
      const int t = s * tp + tl;
      if (rows_s) rows_s[t * k + jl] = row;
      if (write) {
        if (a.row_of) a.row_of[(size_t)t * k + jl] = row;
        if (a.token_of_row && row >= 0) a.token_of_row[row] = t;
      }
    }
  };
  if (hold) {
#pragma unroll
    for (int b = 0; b < kHold; ++b) {
      if (b >= per) break;
      place(s0 + b, held[b]);
    }
  } else {
    for (int s = s0; s < s1; s += kHold) {
#pragma unroll
      for (int b = 0; b < kHold; ++b) held[b] = load(s + b);
#pragma unroll
      for (int b = 0; b < kHold; ++b) place(s + b, pack(held[b]));
    }
  }
}

inline size_t sort_smem(int E) { return sizeof(int) * ((size_t)kSortWarps * E + 2 * (size_t)E + 32); }

__global__ void __launch_bounds__(kSortThreads)
sort_kernel(const SortArgs a) {
  extern __shared__ int sort_smem_raw[];
  cg::cluster_group cl = cg::this_cluster();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the copy may load x meanwhile
  sort_pairs<0>(a, (int)cl.block_rank(), (int)cl.num_blocks(), sort_smem_raw, true, nullptr);
  // the last remote reads happened before the base scan's barriers of each
  // CTA; wait for the cluster so that no CTA leaves while its totals are read
  cl.sync();
}

// Many pairs: CTAs count their shares, one CTA turns the counts into first rows, and
// the CTAs count again (beside the first two launches) and place their pairs.
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const SortArgs a) {
  extern __shared__ int sort_smem_raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  sort_pairs<1>(a, (int)blockIdx.x, (int)gridDim.x, sort_smem_raw, true, nullptr);
}

__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const SortArgs a) {
  extern __shared__ int sort_smem_raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  sort_pairs<2>(a, (int)blockIdx.x, (int)gridDim.x, sort_smem_raw, true, nullptr);
}

// counts of (CTA, expert) -> first rows.  1024 / E groups of threads take runs of
// CTAs; a thread holds its run's counts of one expert.
__global__ void __launch_bounds__(kSortThreads)
sort_first_kernel(const SortArgs a, int ctas) {
  __shared__ int sums[kSortThreads], warp_sums[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int E = a.E, groups = kSortThreads / E, g = threadIdx.x / E, e = threadIdx.x % E;
  const int run = (ctas + groups - 1) / groups, c0 = min(ctas, g * run), c1 = g < groups ? min(ctas, c0 + run) : c0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int n = 0;
#pragma unroll 8
  for (int c = c0; c < c1; ++c) {
    int v;
    asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(v) : "l"(wide_counts(a, c, ctas) + e));
    n += v;
  }
  if (g < groups) sums[threadIdx.x] = n;
  __syncthreads();
  int all = 0, before = 0;
  for (int q = 0; q < groups; ++q) {
    const int v = g < groups ? sums[q * E + e] : 0;
    if (q < g) before += v;
    all += v;
  }
  // experts' first rows: a scan over the threads of group 0
  int incl = g == 0 ? all : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(kFull, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int v = warp_sums[lane];
    int si = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(kFull, si, d);
      if (lane >= d) si += o;
    }
    warp_sums[lane] = si - v;
  }
  __syncthreads();
  if (g == 0) {
    const int first = warp_sums[warp] + incl - all;
    a.offsets[e] = first;
    if (e == E - 1) a.offsets[E] = first + all;
    sums[e] = first;                                   // sums have been read
  }
  __syncthreads();
  if (g < groups) {
    int at = sums[e] + before;
#pragma unroll 8
    for (int c = c0; c < c1; ++c) {
      int32_t* p = wide_counts(a, c, ctas) + e;
      int v;
      asm volatile("ld.global.cg.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
      *p = c == ctas - 1 ? all : at;                   // the last CTA's place is the output `counts`
      at += v;
    }
  }
}

// Every CTA sorts all pairs and copies the rows of its own share of the
// 16-byte vectors; CTA 0 writes the index outputs.  A token's slots are split in as
// many groups as fill the SMs: one SM stores 64 bytes a cycle, so 8 copies of 1024
// vectors from one CTA would take 1 us.
__global__ void __launch_bounds__(kSortThreads)
sort_gather_kernel(const SortArgs a, const uint4* __restrict__ x, int vec, int groups, int per,
                   uint4* __restrict__ xp) {
  extern __shared__ int sort_smem_raw[];
  int32_t* rows_s = sort_smem_raw + kSortWarps * a.E + 2 * a.E + 32;
  const int total = a.T * groups * vec;                // the fused launch is small
  int i = (int)threadIdx.x < per ? (int)(blockIdx.x * per + threadIdx.x) : total;
  int q = i / vec, c = i - q * vec, t = q / groups;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (i < total) v = __ldg(x + t * vec + c);           // in flight while the pairs are sorted
  sort_pairs<0>(a, 0, 1, sort_smem_raw, blockIdx.x == 0, rows_s);
  __syncthreads();
  while (i < total) {
    for (int j = q - t * groups; j < a.k; j += groups) {
      const int r = rows_s[t * a.k + j];
      if (r >= 0) xp[(size_t)r * vec + c] = v;
    }
    i += gridDim.x * per;
    if (i >= total) break;
    q = i / vec, c = i - q * vec, t = q / groups;
    v = __ldg(x + t * vec + c);
  }
}

// xp[row_of[t, j]] = x[t] and token_of_row[row_of[t, j]] = t for every slot j with
// a row (the latter is one 4-byte store per row wherever it lands: a cluster's
// few SMs took 6 us for 98 thousand, here they ride along).  A dependent launch: x
// was complete before the sort began, so its loads do not wait for the sort.
__global__ void __launch_bounds__(kThreads)
scatter_rows_kernel(const uint4* __restrict__ x, int T, int vec, int k, const int32_t* __restrict__ row_of,
                    uint4* __restrict__ xp, int max_rows, int32_t* __restrict__ token_of_row) {
  const size_t first = (size_t)blockIdx.x * kThreads;
  const unsigned rem = (unsigned)(first % vec) + threadIdx.x;
  const size_t t = first / vec + rem / vec;
  const unsigned c = rem % vec;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (t < (size_t)T) v = __ldcs(x + t * vec + c);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (t >= (size_t)T) return;
  for (int j0 = 0; j0 < k; j0 += 4) {
    int r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {                      // asm: stays behind the wait
      r[j] = -1;
      if (j0 + j < k) asm volatile("ld.global.b32 %0, [%1];" : "=r"(r[j]) : "l"(row_of + t * k + j0 + j) : "memory");
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((unsigned)r[j] < (unsigned)max_rows) {
        __stcs(xp + (size_t)r[j] * vec + c, v);
        if (c == 0 && token_of_row) token_of_row[r[j]] = (int)t;
      }
  }
}

// dst[r] = src[index[r]], 16 bytes per thread and step.
__global__ void __launch_bounds__(kThreads)
gather_rows_kernel(const uint4* __restrict__ src, const int32_t* __restrict__ index, int rows, int vec,
                   uint4* __restrict__ dst) {
  const size_t total = (size_t)rows * vec;
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const size_t r = i / vec;
    const int c = (int)(i % vec);
    dst[r * vec + c] = __ldg(src + (size_t)__ldg(index + r) * vec + c);
  }
}

// A launch that may begin when the CTAs of the one before it say so.
template <class... P, class... Q>
zmoe_status launch_dependent(const char* what, void (*kernel)(P...), int ctas, size_t smem, cudaStream_t stream, Q... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, kernel, args...));
  return launch_status(what);
}

zmoe_status launch_sort_wide(const SortArgs& a, int ctas, cudaStream_t stream) {
  zmoe_status st = allow_smem<sort_count_kernel>();
  if (st == ZMOE_OK) st = allow_smem<sort_place_kernel>();
  if (st != ZMOE_OK) return st;
  const size_t smem = sort_smem(a.E);
  sort_count_kernel<<<ctas, kSortThreads, smem, stream>>>(a);
  st = launch_status("sort_count_kernel");
  if (st == ZMOE_OK) st = launch_dependent("sort_first_kernel", sort_first_kernel, 1, 0, stream, a, ctas);
  if (st == ZMOE_OK) st = launch_dependent("sort_place_kernel", sort_place_kernel, ctas, smem, stream, a);
  return st;
}

// One CTA while each of its warps has one step at most, else the largest cluster
// (64 groups, one against 16 CTAs, us: 512 pairs 4.9 and 5.4, 1024 pairs 5.6 and
// 6.2, 2048 pairs 6.9 and 6.3, 16384 pairs 25 and 6.4; 8 CTAs 7.7, 4 CTAs 10.2).
zmoe_status launch_sort(const SortArgs& a, cudaStream_t stream) {
  const size_t smem = sort_smem(a.E);
  zmoe_status st = allow_smem<sort_kernel>();
  if (st != ZMOE_OK) return st;
  static std::atomic<uint64_t> wide{0};                // devices on which the kernel may use 16-CTA clusters
  int dev = 0;
  ZMOE_CUDA_RET(cudaGetDevice(&dev));
  if (!(wide.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    ZMOE_CUDA_RET(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    wide.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const int tp = 32 / a.k, steps = (a.T + tp - 1) / tp;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(steps <= kSortWarps ? 1 : kSortCluster);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cfg.gridDim.x;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, sort_kernel, a));
  return launch_status("sort_kernel");
}

// The form a call takes, by its sizes alone.
struct Plan {
  enum Form { kNothing, kFused, kCluster, kWide, kRanked } form;
  bool copy;                                           // a launch of its own for the rows
  int per;                                             // kWide: steps per warp
  int launches() const {
    const int sort[] = {0, 1, 1, 3, 2};
    return sort[form] + (copy ? 1 : 0);
  }
};
Plan plan_of(const zmoe_permute_args* a) {
  const int vec = a->H / 8;
  Plan p{Plan::kNothing, false, 0};
  if (a->T <= 0) return p;
  p.copy = a->xp != nullptr && vec > 0;
  p.form = Plan::kRanked;
  if (a->capacity > 0 || a->E > kSortE || a->k > 32) return p;
  p.form = Plan::kCluster;
  const long long pairs = (long long)a->T * a->k;
  if (p.copy && pairs <= kFusedPairs && (long long)a->T * vec < 1 << 30) {
    p.form = Plan::kFused;
    p.copy = false;
    return p;
  }
  const int tp = 32 / a->k, steps = (int)(((long long)a->T + tp - 1) / tp);
  const int per = (steps + kWideCtas * kSortWarps - 1) / (kWideCtas * kSortWarps);
  if (pairs >= kWidePairs && kSortWarps * per * tp * a->k >= a->E) {
    p.form = Plan::kWide;
    p.per = per;
  }
  return p;
}

}  // namespace

int permute_launches(const zmoe_permute_args* a) { return plan_of(a).launches(); }

zmoe_status launch_permute(const zmoe_permute_args* a, cudaStream_t stream) {
  ZMOE_CHECK_ARG(a && a->topk_idx && a->counts && a->offsets && a->row_of && a->token_of_row,
                 "permute: null pointer");
  ZMOE_CHECK_ARG(a->E >= 1 && a->k >= 1, "permute: bad E/k");
  ZMOE_CHECK_ARG(a->capacity <= 0 || (a->seq_len > 0 && a->T % a->seq_len == 0),
                 "permute: T=%d must be a multiple of seq_len=%d when capacity is set", a->T, a->seq_len);
  ZMOE_CHECK_ARG(a->xp == nullptr || (a->x && a->H % 8 == 0 && (uintptr_t)a->x % 16 == 0 && (uintptr_t)a->xp % 16 == 0),
                 "permute: gather needs H %% 8 == 0 and 16-byte aligned x/xp");
  if (a->T <= 0) {
    ZMOE_CUDA_RET(cudaMemsetAsync(a->counts, 0, sizeof(int32_t) * a->E, stream));
    ZMOE_CUDA_RET(cudaMemsetAsync(a->offsets, 0, sizeof(int32_t) * (a->E + 1), stream));
    return ZMOE_OK;
  }
  ZMOE_CHECK_ARG(a->T <= kMaxT && (long long)a->T * a->k < (1LL << 31), "permute: T=%d x k=%d pairs are too many", a->T, a->k);
  const int vec = a->H / 8;
  const Plan plan = plan_of(a);
  const size_t blocks = ((size_t)a->T * vec + kThreads - 1) / kThreads;
  ZMOE_CHECK_ARG(!plan.copy || blocks < ((size_t)1 << 31), "permute: T=%d rows of H=%d are too many for one launch", a->T, a->H);
  zmoe_status st;
  if (plan.form == Plan::kRanked) {
    ZMOE_CUDA_RET(cudaMemsetAsync(a->row_of, 0xff, sizeof(int32_t) * (size_t)a->T * a->k, stream));
    count_kernel<<<a->E, kThreads, 0, stream>>>(a->topk_idx, a->T, a->k, a->capacity, a->seq_len, a->counts);
    st = launch_status("count_kernel");
    if (st != ZMOE_OK) return st;
    scatter_kernel<<<a->E, kThreads, 0, stream>>>(a->topk_idx, a->T, a->k, a->E, a->counts, a->offsets,
                                                  a->row_of, a->token_of_row);
    st = launch_status("scatter_kernel");
  } else {
    // behind a sort the copy of the rows writes token_of_row
    const SortArgs sa{a->topk_idx, a->T, a->k, a->E, 0, a->counts, a->offsets, a->row_of,
                      plan.copy ? nullptr : a->token_of_row, plan.per};
    const int tp = 32 / a->k, steps = (a->T + tp - 1) / tp;
    if (plan.form == Plan::kFused) {
      st = allow_smem<sort_gather_kernel>();
      if (st != ZMOE_OK) return st;
      const size_t smem = sort_smem(a->E) + sizeof(int32_t) * (size_t)a->T * a->k;
      const int full = kNumSMs * kSortThreads / (a->T * vec);
      const int groups = full < 1 ? 1 : full < a->k ? full : a->k;
      const int items = a->T * groups * vec;
      int per = (items / kNumSMs + 255) / 256 * 256;   // of a CTA at a time
      per = per < 256 ? 256 : per > kSortThreads ? kSortThreads : per;
      int ctas = (items + per - 1) / per;
      if (ctas > kNumSMs) ctas = kNumSMs;
      sort_gather_kernel<<<ctas, kSortThreads, smem, stream>>>(sa, reinterpret_cast<const uint4*>(a->x), vec, groups, per,
                                                               reinterpret_cast<uint4*>(a->xp));
      return launch_status("sort_gather_kernel");
    }
    st = plan.form == Plan::kWide ? launch_sort_wide(sa, (steps + kSortWarps * plan.per - 1) / (kSortWarps * plan.per), stream)
                                  : launch_sort(sa, stream);
  }
  if (st != ZMOE_OK || !plan.copy) return st;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  ZMOE_CUDA_RET(cudaLaunchKernelEx(&cfg, scatter_rows_kernel, reinterpret_cast<const uint4*>(a->x), a->T, vec, a->k,
                                   (const int32_t*)a->row_of, reinterpret_cast<uint4*>(a->xp), a->T * a->k,
                                   plan.form == Plan::kRanked ? (int32_t*)nullptr : a->token_of_row));
  return launch_status("scatter_rows_kernel");
}

zmoe_status launch_lora_plan(const int32_t* adapter, int T, int G, int32_t* offsets, int32_t* token_of_row,
                             cudaStream_t stream) {
  ZMOE_CHECK_ARG(G >= 1 && G < kSortE, "lora_plan: G=%d outside [1, %d]", G, kSortE - 1);
  ZMOE_CHECK_ARG(T >= 0 && offsets && (T == 0 || (adapter && token_of_row)), "lora_plan: null pointer or negative T");
  ZMOE_CHECK_ARG(T <= kMaxT, "lora_plan: T=%d above %d", T, kMaxT);
  const Span w[] = {{"offsets", offsets, 4 * ((size_t)G + 1)}, {"token_of_row", T ? token_of_row : nullptr, 4 * (size_t)T}};
  const Span r[] = {{"adapter", T ? adapter : nullptr, 4 * (size_t)T}};
  const char *p, *q;
  ZMOE_CHECK_ARG(apart(w, r, &p, &q), "lora_plan: %s must not overlap %s", p, q);
  if (T == 0) {
    ZMOE_CUDA_RET(cudaMemsetAsync(offsets, 0, sizeof(int32_t) * (size_t)(G + 1), stream));
    return ZMOE_OK;
  }
  return launch_sort(SortArgs{adapter, T, 1, G + 1, 1, nullptr, offsets, nullptr, token_of_row, 0}, stream);
}

zmoe_status launch_gather_rows(const void* src, const int32_t* index, int rows, int row_bytes, void* dst,
                               cudaStream_t stream) {
  ZMOE_CHECK_ARG(rows >= 0 && row_bytes > 0 && row_bytes % 16 == 0, "gather_rows: rows=%d, row_bytes=%d (multiple of 16)",
                 rows, row_bytes);
  if (rows == 0) return ZMOE_OK;
  ZMOE_CHECK_ARG(src && index && dst && (uintptr_t)src % 16 == 0 && (uintptr_t)dst % 16 == 0,
                 "gather_rows: null or unaligned pointer");
  const int vec = row_bytes / 16;
  size_t blocks = ((size_t)rows * vec + kThreads - 1) / kThreads;
  if (blocks > (size_t)kNumSMs * 8) blocks = (size_t)kNumSMs * 8;
  gather_rows_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(static_cast<const uint4*>(src), index, rows, vec,
                                                                static_cast<uint4*>(dst));
  return launch_status("gather_rows_kernel");
}

}  // namespace zmoe
