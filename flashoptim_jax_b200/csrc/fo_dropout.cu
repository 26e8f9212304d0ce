// Dropout from a counter-based generator, with an optional residual:  y = residual + x * keep / (1 - p).
// The mask is a function of (seed, offset, element) and is never stored: the backward pass is the same call on the gradient.
#include "fo_tokens.cuh"

namespace fo {

constexpr int kDropThreads = 256;
constexpr int kDropOcts = 2;  // per thread, a block's width apart, all loads in flight before the first is used

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

// Bound by HBM: n elements read (twice with a residual) and written, 16 bytes at a time.  Calls in a graph, where part of a result stays in the L2 until the next call: 67 M bf16 elements
// 45 us (40 with p = 0, without the draws), with a residual 58, 16 M fp32 elements 18 to 19; as calls of their own 65 (6.2 TB/s) and 20.8 (6.1).  A draw keeps the multiply pipe busy for 80 cycles a warp: drawn before the loaded
// elements are touched, it hides behind them (drawn after: 59, 78 and 22 us).  A launch of as many blocks as there is work, two blocks of eight elements a
// thread: with one 67 us without a residual and p = 0, with four as long and more registers.
template <int DT, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const __grid_constant__ DropoutParams p) {
  chain_wait();
  chain_release();
  const Drop& d = p.drop;
  const uint2 off = drop_offset(d);
  constexpr int kBytes = 8 * size_of(DT);
  const unsigned long long octs = p.n / 8;
  const unsigned long long q0 = (unsigned long long)blockIdx.x * kDropThreads * kDropOcts + threadIdx.x;
  if (q0 < octs) {
    Oct<DT> x[kDropOcts], r[kDropOcts];
#pragma unroll
    for (int k = 0; k < kDropOcts; ++k) {
      const unsigned long long q = q0 + k * kDropThreads;
      if (q < octs) {
        x[k].load((const char*)p.x + q * kBytes);
        if constexpr (RES) r[k].load((const char*)p.residual + q * kBytes);
      }
    }
    uint4 w[kDropOcts];  // drawn while the elements are on their way
    if (d.on) {
#pragma unroll
      for (int k = 0; k < kDropOcts; ++k) w[k] = draw8(d, off, q0 + k * kDropThreads);
    }
#pragma unroll
    for (int k = 0; k < kDropOcts; ++k) {
      const unsigned long long q = q0 + k * kDropThreads;
      if (q >= octs) break;
      float v[8], a[8];
      x[k].get(v);
      if constexpr (RES) r[k].get(a);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmul(v[j], p.factor);
      if (d.on) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = stays(d, w[k], j) ? v[j] : 0.0f;
      }
      if constexpr (RES) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fadd(a[j], v[j]);
      }
      x[k].set(v);
      x[k].store((char*)p.y + q * kBytes);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (p.n & 7)) {  // the ragged end
    const unsigned long long i = octs * 8 + threadIdx.x;
    const bool keep = !d.on || (keep8(d, off, octs) >> threadIdx.x & 1u) != 0;
    float r = 0.0f;
    if constexpr (RES) r = load1<DT>(p.residual, i);
    store1<DT>(p.y, i, dropped<DT, RES>(load1<DT>(p.x, i), r, keep, p.factor));
  }
}

// Arrays that are not aligned: 256 elements per warp, neighbours in neighbouring lanes, each lane drawing eight neighbours and handing them on.
template <int DT, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_unaligned_kernel(const __grid_constant__ DropoutParams p) {
  chain_wait();
  chain_release();
  const Drop& d = p.drop;
  const uint2 off = drop_offset(d);
  const int lane = threadIdx.x & 31;
  const unsigned long long first = ((unsigned long long)blockIdx.x * kDropThreads + (threadIdx.x & ~31u)) * 8;
  float x[8], r[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned long long i = first + j * 32 + lane;
    if (i < p.n) {
      x[j] = load1<DT>(p.x, i);
      if constexpr (RES) r[j] = load1<DT>(p.residual, i);
    }
  }
  const uint32_t mine = d.on ? keep8(d, off, first / 8 + lane) : 0xFFu;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool keep = (__shfl_sync(~0u, mine, j * 4 + lane / 8) >> (lane & 7) & 1u) != 0;
    if (first + j * 32 + lane < p.n) store1<DT>(p.y, first + j * 32 + lane, dropped<DT, RES>(x[j], r[j], keep, p.factor));
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
  p.x = x; p.residual = residual; p.y = y; p.n = n; p.factor = (float)factor;
  const bool aligned = on_16_bytes(x) && on_16_bytes(residual) && on_16_bytes(y);
  const unsigned long long per_block = (unsigned long long)kDropThreads * 8 * (aligned ? kDropOcts : 1);
  const unsigned long long blocks = (n + per_block - 1) / per_block;
  if (blocks > 0x7FFFFFFFull) return fail(FO_ERR_TOO_LARGE, "fo_dropout: %llu elements exceed one launch", (unsigned long long)n);
  void (*kernel)(const DropoutParams) = nullptr;
#define X(D)                                                                                                        \
  if (dtype == D) kernel = residual != nullptr ? (aligned ? dropout_kernel<D, true> : dropout_unaligned_kernel<D, true>) \
                                               : (aligned ? dropout_kernel<D, false> : dropout_unaligned_kernel<D, false>);
  X(FO_F32) X(FO_BF16) X(FO_F16)
#undef X
  bool chained = true;
  const cudaError_t e = launch_chained(kernel, (unsigned int)blocks, (unsigned int)kDropThreads, 0, chained, (cudaStream_t)stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_dropout: launch failed: %s", cudaGetErrorString(e));
}
