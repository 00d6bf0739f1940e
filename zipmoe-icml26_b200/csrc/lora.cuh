// Shared by the adapter kernels: units of work from the row groups, and small helpers.
#pragma once
#include "common.cuh"

namespace zmoe {
namespace lora {

constexpr int kThreads = 256;
constexpr int kMaxCols = 32768;                        // H and N
constexpr int kMaxT = 1 << 30;                         // row and tile indexes are int
constexpr unsigned kFull = 0xffffffffu;
constexpr int kAhead = 4;                              // of find_unit

// lora_tc.cu
zmoe_status launch_tiles(const zmoe_lora_args* a, cudaStream_t stream);
zmoe_status launch_grad_tiles(const zmoe_lora_grad_args* a, cudaStream_t stream);
zmoe_status read_error(int32_t* out, int reset);

// Up to `tile` consecutive rows of one group; g >= G: rows without adapter.
struct Unit {
  int g, row0, rows;                                   // rows == 0: no such unit
};

// Unit u of the groups' tiles, in order; `rest`: the rows behind the last
// group, and those before the first, are groups too.  Called by one full warp; offsets are clamped to
// [0, T], so a unit never reaches past the last row.
__device__ __forceinline__ Unit find_unit(const int32_t* __restrict__ offsets, int G, int T, int tile, bool rest, int u) {
  const int lane = threadIdx.x & 31;
  const int groups = G + (rest ? 2 : 0);
  int before = 0;
  for (int g0 = 0; g0 < groups; g0 += 32 * kAhead) {
    int r0[kAhead], n[kAhead];                         // kAhead warps of groups, loaded together
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int g = g0 + 32 * i + lane;
      r0[i] = n[i] = 0;
      if (g < groups) {
        r0[i] = g <= G ? min(max(__ldg(offsets + g), 0), T) : 0;
        const int r1 = g == G ? T : min(max(__ldg(offsets + (g < G ? g + 1 : 0)), 0), T);
        n[i] = max(0, r1 - r0[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int tiles = (n[i] + tile - 1) / tile;
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += o;
      }
      const int first = before + incl - tiles;
      const unsigned hit = __ballot_sync(kFull, u >= first && u < first + tiles);
      if (hit) {
        const int src = __ffs(hit) - 1;
        const int local = u - __shfl_sync(kFull, first, src);
        const int gr0 = __shfl_sync(kFull, r0[i], src), gn = __shfl_sync(kFull, n[i], src);
        return Unit{g0 + 32 * i + src, gr0 + local * tile, min(tile, gn - local * tile)};
      }
      before += __shfl_sync(kFull, incl, 31);
      if (g0 + 32 * (i + 1) >= groups) break;
    }
  }
  return Unit{0, 0, 0};
}

// Token of a row, -1 when the list names none.
__device__ __forceinline__ int token_of(const int32_t* token_of_row, int row, int T) {
  const int t = token_of_row ? __ldg(token_of_row + row) : row;
  return (unsigned)t < (unsigned)T ? t : -1;
}

// Columns of one of `parts` slices of n columns, in whole 16-byte vectors.
__host__ __device__ __forceinline__ int slice8(int n, int parts) { return (n / 8 + parts - 1) / parts * 8; }

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f[2 * q] = __uint_as_float(w[q] << 16);
    f[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
  }
}

// A value as three BF16 terms (the upper halves of t) whose sum it is: each is what
// the ones before leave, cut to 8 bits.  Infinities and NaN are their first term.
__device__ __forceinline__ void split(float f, uint32_t (&t)[3]) {
  const uint32_t b = __float_as_uint(f);
  const bool finite = (b & 0x7f800000u) != 0x7f800000u;
  const float rest = finite ? f - __uint_as_float(b & 0xffff0000u) : 0.0f;
  t[0] = finite || !(b & 0x007fffffu) ? b : b | 0x00400000u;   // a NaN stays one
  t[1] = __float_as_uint(rest);
  t[2] = __float_as_uint(rest - __uint_as_float(t[1] & 0xffff0000u));
}

// Eight values as three vectors of BF16 terms.
__device__ __forceinline__ void split8(const float4 (&f)[2], uint4 (&t)[3]) {
  const float v[8] = {f[0].x, f[0].y, f[0].z, f[0].w, f[1].x, f[1].y, f[1].z, f[1].w};
  uint32_t w[3][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t a[3], b[3];
    split(v[2 * q], a);
    split(v[2 * q + 1], b);
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i][q] = __byte_perm(a[i], b[i], 0x7632);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) t[i] = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

}  // namespace lora
}  // namespace zmoe
