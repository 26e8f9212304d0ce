// Dropout from a counter-based generator, with an optional residual:  y = residual + x * keep / (1 - p).
// The mask is a function of (seed, offset, element) and is never stored: the backward pass is the same call on the gradient.
#include "fo_tokens.cuh"

namespace fo {

constexpr int kDropThreads = 256;
constexpr int kDropOcts = 4;  // per thread, a block's width apart, all loads in flight before the first is used

struct DropoutParams {
  const void* x;
  const void* residual;
  void* y;
  unsigned long long n;
  float factor;  // 1 / (1 - p)
  Drop drop;
};

// A dropped element is 0 whatever it held.
template <int DT, bool RES>
FO_DEVI float dropped(const float x, const float r, const bool keep, const float factor) {
  const float v = keep ? fmul(x, factor) : 0.0f;
  return RES ? fadd(r, v) : v;
}

// Bound by HBM: n elements read (twice with a residual) and written.  Whole blocks of eight elements, 16-byte accesses.
template <int DT, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  chain_wait();
  chain_release();
  Drop d = p.drop;
  resolve_offset(d);
  constexpr int kBytes = 8 * size_of(DT);
  const unsigned long long octs = p.n / 8;
  const unsigned long long step = (unsigned long long)gridDim.x * kDropThreads * kDropOcts;
  for (unsigned long long q0 = (unsigned long long)blockIdx.x * kDropThreads * kDropOcts + threadIdx.x; q0 < octs; q0 += step) {
    Oct<DT> x[kDropOcts], r[kDropOcts];
#pragma unroll
    for (int k = 0; k < kDropOcts; ++k) {
      const unsigned long long q = q0 + k * kDropThreads;
      if (q < octs) {
        x[k].load((const char*)p.x + q * kBytes);
        if constexpr (RES) r[k].load((const char*)p.residual + q * kBytes);
      }
    }
#pragma unroll
    for (int k = 0; k < kDropOcts; ++k) {
      const unsigned long long q = q0 + k * kDropThreads;
      if (q >= octs) break;
      const uint32_t keep = d.on ? keep8(d, q) : 0xFFu;
      float v[8], a[8];
      x[k].get(v);
      if constexpr (RES) r[k].get(a);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = dropped<DT, RES>(v[j], RES ? a[j] : 0.0f, (keep >> j & 1u) != 0, p.factor);
      x[k].set(v);
      x[k].store((char*)p.y + q * kBytes);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (p.n & 7)) {  // the ragged end
    const unsigned long long i = octs * 8 + threadIdx.x;
    const bool keep = !d.on || (keep8(d, octs) >> threadIdx.x & 1u) != 0;
    float r = 0.0f;
    if constexpr (RES) r = load1<DT>(p.residual, i);
    store1<DT>(p.y, i, dropped<DT, RES>(load1<DT>(p.x, i), r, keep, p.factor));
  }
}

// Arrays that are not aligned: eight elements per thread, one at a time.
template <int DT, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_unaligned_kernel(const __grid_constant__ DropoutParams p) {
  chain_wait();
  chain_release();
  Drop d = p.drop;
  resolve_offset(d);
  const unsigned long long octs = (p.n + 7) / 8;
  for (unsigned long long q = (unsigned long long)blockIdx.x * kDropThreads + threadIdx.x; q < octs; q += (unsigned long long)gridDim.x * kDropThreads) {
    const uint32_t keep = d.on ? keep8(d, q) : 0xFFu;
    float x[8], r[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long i = q * 8 + j;
      if (i < p.n) {
        x[j] = load1<DT>(p.x, i);
        if constexpr (RES) r[j] = load1<DT>(p.residual, i);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (q * 8 + j < p.n) store1<DT>(p.y, q * 8 + j, dropped<DT, RES>(x[j], r[j], (keep >> j & 1u) != 0, p.factor));
  }
}

}  // namespace fo

using namespace fo;

extern "C" int fo_dropout(const void* x, const void* residual, void* y, int32_t dtype, uint64_t n, const FoDropout* dropout, void* stream) {
  if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARG, "fo_dropout: bad dtype %d", dtype);
  DropoutParams p;
  double factor;
  if (dropout == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_dropout: null dropout");
  if (!make_drop(dropout, p.drop, factor)) return fail(FO_ERR_INVALID_ARG, "fo_dropout: p = %g (it lies in [0, 1]), dev_offset_bits = %d (32 or 64)", dropout->p, dropout->dev_offset_bits);
  if (n == 0) return FO_OK;
  if (x == nullptr || y == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_dropout: null pointer");
  if (n >> 60) return fail(FO_ERR_TOO_LARGE, "fo_dropout: %llu elements", (unsigned long long)n);
  p.x = x; p.residual = residual; p.y = y; p.n = n; p.factor = (float)factor;
  const bool aligned = on_16_bytes(x) && on_16_bytes(residual) && on_16_bytes(y);
  const unsigned long long per_block = (unsigned long long)kDropThreads * 8 * (aligned ? kDropOcts : 1);
  const unsigned long long blocks = (n + per_block - 1) / per_block;
  const unsigned int grid = (unsigned int)(blocks < 0x7FFFFFFFull ? blocks : 0x7FFFFFFFull);
  void (*kernel)(const DropoutParams) = nullptr;
#define X(D)                                                                                                        \
  if (dtype == D) kernel = residual != nullptr ? (aligned ? dropout_kernel<D, true> : dropout_unaligned_kernel<D, true>) \
                                               : (aligned ? dropout_kernel<D, false> : dropout_unaligned_kernel<D, false>);
  X(FO_F32) X(FO_BF16) X(FO_F16)
#undef X
  bool chained = true;
  const cudaError_t e = launch_chained(kernel, grid, (unsigned int)kDropThreads, 0, chained, (cudaStream_t)stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_dropout: launch failed: %s", cudaGetErrorString(e));
}
