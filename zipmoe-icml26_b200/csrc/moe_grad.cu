// Gradients of the permute and the combine.
//
//   permute:  xp[row_of[t, j]] = x[t]             dx[t] = base[t] + sum_j dxp[row_of[t, j]]
//   combine:  out[t] = sum_j w[t, j] y[row] + g[t] ysh[t]
//             dy[row] = w[t, j] dout[t]           dw[t, j] = <dout[t], y[row]>
//             dysh[t] = g[t] dout[t]              dg[t] = <dout[t], ysh[t]>
// A row belongs to one (token, slot) pair, so every output element has one
// writer: sums run over a token's slots in slot order in fp32, dot products
// over a fixed order of lanes, and each output is rounded once.  Both kernels
// are bound by HBM: they read and write every row once.
#include "common.cuh"

namespace zmoe {
namespace {

constexpr int kThreads = 256;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f[2 * q] = __uint_as_float(w[q] << 16);
    f[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    w[q] = (uint32_t)f32_to_bf16_bits(f[2 * q]) | ((uint32_t)f32_to_bf16_bits(f[2 * q + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One 16-byte vector of one token per thread; the slots' loads are issued
// kSlots at a time before their sum.  kSlots is k itself up to 8: registers for
// slots that are not there cost loads in flight (16383 tokens of 6 rows of 2048
// with a base: 95 us with room for 8 slots, 86 us, 6.2 TB/s, with 6).
template <int kSlots>
__global__ void __launch_bounds__(kThreads)
permute_grad_kernel(const uint4* __restrict__ dxp, const int32_t* __restrict__ row_of, const uint4* base, int T,
                    int vec, int k, int rows, uint4* dx) {
  const size_t first = (size_t)blockIdx.x * kThreads;
  const unsigned rem = (unsigned)(first % vec) + threadIdx.x;
  const size_t t = first / vec + rem / vec;
  const unsigned c = rem % vec;
  if (t >= (size_t)T) return;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  uint4 b = make_uint4(0, 0, 0, 0);
  if (base) b = __ldcs(base + t * vec + c);
  for (int j0 = 0; j0 < k; j0 += kSlots) {
    uint4 v[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = j0 + j < k ? __ldg(row_of + t * k + j0 + j) : -1;
      v[j] = make_uint4(0, 0, 0, 0);
      if ((unsigned)r < (unsigned)rows) v[j] = __ldcs(dxp + (size_t)r * vec + c);
    }
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j0 + j >= k) break;
      float f[8];
      unpack8(v[j], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += f[i];
    }
  }
  if (base) {
    float f[8];
    unpack8(b, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += f[i];
  }
  __stcs(dx + t * vec + c, pack8(acc));
}

// One warp per (token, slot), the shared expert as slot k: it reads dout[t] and
// the slot's row, writes the scaled row and keeps the dot product.  A token's
// slots are neighbouring warps, so dout comes from L1 for all but the first.
// (A warp per token that held dout in registers would read it once, but runs
// the slots one after another: too few loads in flight for short batches.)
constexpr int kUnroll = 4;

__global__ void __launch_bounds__(kThreads)
combine_grad_kernel(const zmoe_combine_grad_args a, int slots) {
  const int lane = threadIdx.x & 31;
  const size_t unit = (size_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const size_t t = unit / (unsigned)slots;
  const int j = (int)(unit % (unsigned)slots);
  if (t >= (size_t)a.T) return;
  const int vec = a.H / 8;
  const uint4* dout = reinterpret_cast<const uint4*>(a.dout) + t * vec;
  const uint4* src = nullptr;                          // the row of the dot product
  uint4* dst = nullptr;                                // the scaled row
  float w = 1.0f;
  bool pass = false;                                   // Switch, dropped: the row is the token's own
  if (j < a.k) {
    const int r = a.row_of[t * a.k + j];
    w = a.topk_w[t * a.k + j];
    if ((unsigned)r < (unsigned)a.rows) {
      src = reinterpret_cast<const uint4*>(a.y) + (size_t)r * vec;
      dst = reinterpret_cast<uint4*>(a.dy) + (size_t)r * vec;
    } else if (a.mode == ZMOE_ROUTE_SWITCH) {
      pass = true;
      src = reinterpret_cast<const uint4*>(a.x) + t * vec;
      dst = reinterpret_cast<uint4*>(a.dx) + t * vec;
    }
  } else {
    if (a.shared_gate) w = a.shared_gate[t];
    if (a.dshared_gate) src = reinterpret_cast<const uint4*>(a.y_shared) + t * vec;
    if (a.dy_shared) dst = reinterpret_cast<uint4*>(a.dy_shared) + t * vec;
  }
  float dot = 0.0f;
  if (src || dst) {
    for (int c0 = lane; c0 < vec; c0 += 32 * kUnroll) {
      uint4 d[kUnroll], v[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int c = c0 + 32 * q;
        d[q] = v[q] = make_uint4(0, 0, 0, 0);
        if (c < vec) {
          d[q] = __ldg(dout + c);
          if (src) v[q] = __ldcs(src + c);
        }
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int c = c0 + 32 * q;
        float df[8], vf[8], s = 0.0f;
        unpack8(d[q], df);
        unpack8(v[q], vf);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s = fmaf(df[i], vf[i], s);
          df[i] *= w;
        }
        dot += s;
        if (dst && c < vec) __stcs(dst + c, pack8(df));
      }
    }
  }
  if (j == 0 && a.mode == ZMOE_ROUTE_SWITCH && !pass) {
    uint4* z = reinterpret_cast<uint4*>(a.dx) + t * vec;
    for (int c = lane; c < vec; c += 32) __stcs(z + c, make_uint4(0, 0, 0, 0));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) dot += __shfl_xor_sync(kFull, dot, off);
  if (lane == 0) {
    if (j < a.k) a.dtopk_w[t * a.k + j] = dot;
    else if (a.dshared_gate) a.dshared_gate[t] = dot;
  }
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

zmoe_status launch_permute_grad(const zmoe_permute_grad_args* a, cudaStream_t stream) {
  ZMOE_CHECK_ARG(a && a->T >= 0 && a->rows >= 0 && a->k >= 1, "permute_grad: null pointer, negative size or k < 1");
  if (a->T == 0) return ZMOE_OK;
  ZMOE_CHECK_ARG(a->row_of && a->dx && (a->rows == 0 || a->dxp), "permute_grad: null pointer");
  ZMOE_CHECK_ARG(a->H > 0 && a->H % 8 == 0, "permute_grad: H=%d must be a positive multiple of 8", a->H);
  ZMOE_CHECK_ARG(aligned16(a->dxp) && aligned16(a->base) && aligned16(a->dx),
                 "permute_grad: rows must be 16-byte aligned");
  {
    const size_t row = 2 * (size_t)a->H, T = a->T;
    const Span w[] = {{"dx", a->dx, T * row, "base"}};
    const Span r[] = {{"dxp", a->dxp, a->rows * row}, {"row_of", a->row_of, 4 * T * a->k}, {"base", a->base, T * row}};
    const char *p, *q;
    ZMOE_CHECK_ARG(apart(w, r, &p, &q), "permute_grad: %s must not overlap %s", p, q);
  }
  const int vec = a->H / 8;
  const size_t blocks = ((size_t)a->T * vec + kThreads - 1) / kThreads;
  ZMOE_CHECK_ARG(blocks < ((size_t)1 << 31), "permute_grad: T=%d rows of H=%d are too many for one launch", a->T, a->H);
  auto kernel = permute_grad_kernel<8>;
  switch (a->k) {
    case 1: kernel = permute_grad_kernel<1>; break;
    case 2: kernel = permute_grad_kernel<2>; break;
    case 3: kernel = permute_grad_kernel<3>; break;
    case 4: kernel = permute_grad_kernel<4>; break;
    case 5: kernel = permute_grad_kernel<5>; break;
    case 6: kernel = permute_grad_kernel<6>; break;
    case 7: kernel = permute_grad_kernel<7>; break;
  }
  kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(
      reinterpret_cast<const uint4*>(a->dxp), a->row_of, reinterpret_cast<const uint4*>(a->base), a->T, vec, a->k,
      a->rows, reinterpret_cast<uint4*>(a->dx));
  return launch_status("permute_grad_kernel");
}

zmoe_status launch_combine_grad(const zmoe_combine_grad_args* a, cudaStream_t stream) {
  ZMOE_CHECK_ARG(a && a->T >= 0 && a->rows >= 0 && a->k >= 1, "combine_grad: null pointer, negative size or k < 1");
  ZMOE_CHECK_ARG(a->mode >= 0 && a->mode <= 2, "combine_grad: bad mode %d", a->mode);
  if (a->T == 0) return ZMOE_OK;
  ZMOE_CHECK_ARG(a->dout && a->row_of && a->topk_w && a->dtopk_w && (a->rows == 0 || (a->y && a->dy)),
                 "combine_grad: null pointer");
  ZMOE_CHECK_ARG(a->mode != ZMOE_ROUTE_SWITCH || (a->k == 1 && a->x && a->dx && !a->dy_shared && !a->dshared_gate),
                 "combine_grad: Switch needs k = 1, x and dx, and has no shared expert");
  ZMOE_CHECK_ARG(!a->dshared_gate || a->y_shared, "combine_grad: dshared_gate needs y_shared");
  ZMOE_CHECK_ARG(a->H > 0 && a->H % 8 == 0, "combine_grad: H=%d must be a positive multiple of 8", a->H);
  ZMOE_CHECK_ARG(aligned16(a->dout) && aligned16(a->y) && aligned16(a->dy) && aligned16(a->y_shared) &&
                     aligned16(a->dy_shared) && aligned16(a->x) && aligned16(a->dx),
                 "combine_grad: rows must be 16-byte aligned");
  {
    // A warp reads a row's elements before it writes them, so an output may take the
    // place of its own operand; dout is read by several.
    const size_t row = 2 * (size_t)a->H, T = a->T;
    const Span w[] = {{"dy", a->dy, a->rows * row, "y"}, {"dtopk_w", a->dtopk_w, 4 * T * a->k, "topk_w"},
                      {"dy_shared", a->dy_shared, T * row, "y_shared"}, {"dshared_gate", a->dshared_gate, 4 * T, "shared_gate"},
                      {"dx", a->dx, T * row, "x"}};
    const Span r[] = {{"dout", a->dout, T * row}, {"y", a->y, a->rows * row}, {"y_shared", a->y_shared, T * row},
                      {"shared_gate", a->shared_gate, 4 * T}, {"row_of", a->row_of, 4 * T * a->k},
                      {"topk_w", a->topk_w, 4 * T * a->k}, {"x", a->x, T * row}};
    const char *p, *q;
    ZMOE_CHECK_ARG(apart(w, r, &p, &q), "combine_grad: %s must not overlap %s", p, q);
  }
  const int slots = a->k + (a->dy_shared || a->dshared_gate ? 1 : 0);
  const size_t blocks = ((size_t)a->T * slots + kThreads / 32 - 1) / (kThreads / 32);
  ZMOE_CHECK_ARG(blocks < ((size_t)1 << 31), "combine_grad: T=%d x k=%d is too many for one launch", a->T, a->k);
  combine_grad_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(*a, slots);
  return launch_status("combine_grad_kernel");
}

}  // namespace zmoe
