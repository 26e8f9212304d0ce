// Shared by the kernels at the token end of a training step (lookup, its gradient, dropout): eight elements at a time as
// fp32, and the counter-based generator behind dropout.
#pragma once

#include <cmath>

#include "fo_step.cuh"

namespace fo {

int fail(int code, const char* fmt, ...);

// ---- which elements stay -----------------------------------------------------------------------------------------
// Element e of a call stays where its uniform 32-bit number u is at least T = round(p 2^32).  The numbers come from
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) with the key `seed` and the
// counter (e / 8, offset): one block of 128 bits gives the upper 16 bits of u to eight neighbouring elements, and only where one
// of those equals T's does a second block (counter with the top bit set) give the lower 16.  So p is exact to 2^-32, and
// an element costs 1/8 of a block: with 32 bits from the first block on, the ten rounds of two wide products
// would cost twice as much, more than the bytes they decide on take at 6.4 TB/s.
struct Drop {
  uint32_t key[20];  // two per round: an operand of an instruction each, where sums of the seed would take registers in every kernel's loop
  uint32_t off0, off1;
  const void* dev_offset;  // added to the offset when it is not null
  int32_t dev_bits;        // 32 or 64
  uint32_t above;          // what a drawn half, shifted up by 16, is greater than where the element stays
  uint32_t hi, lo;         // T, its upper half in both halves of a word; lo is 0 or a tie needs the second block
  int32_t on;
};

// false: an argument that is none
inline bool make_drop(const FoDropout* f, Drop& d, double& factor) {
  d = Drop{};
  factor = 1.0;
  if (f == nullptr) return true;
  if (!(f->p >= 0.0 && f->p <= 1.0)) return false;
  if (f->dev_offset != nullptr && f->dev_offset_bits != 32 && f->dev_offset_bits != 64) return false;
  const uint64_t t = (uint64_t)(f->p * 4294967296.0 + 0.5);
  if (t == 0) return true;
  d.on = 1;
  for (uint32_t r = 0; r < 10; ++r) {
    d.key[2 * r] = (uint32_t)f->seed + r * 0x9E3779B9u;
    d.key[2 * r + 1] = (uint32_t)(f->seed >> 32) + r * 0xBB67AE85u;
  }
  d.off0 = (uint32_t)f->offset; d.off1 = (uint32_t)(f->offset >> 32);
  d.dev_offset = f->dev_offset; d.dev_bits = f->dev_offset_bits;
  const uint32_t hi = (uint32_t)(t >> 16);
  d.lo = (uint32_t)(t & 0xFFFF);
  d.hi = hi | hi << 16;                                                  // (p = 1: lo is 0, not looked at)
  d.above = (uint32_t)(((uint64_t)hi + (d.lo != 0 && hi != 0xFFFFu ? 1u : 0u)) << 16) - 1u;  // (p = 1: all ones, none stays)
  factor = f->p < 1.0 ? 1.0 / (1.0 - f->p) : 0.0;
  return true;
}

// What elements that stay are multiplied by.  false: neither 0 nor a normal fp32 number (a subnormal one holds too few bits of the product)
inline bool make_factor(const double scale, const double factor, float& out) {
  out = (float)(scale * factor);
  return scale * factor == 0.0 ? scale == 0.0 || factor == 0.0 : std::isnormal(out);
}

// the call's offset, part of which may lie on the device (so that a captured call drops other elements at each replay)
FO_DEVI uint2 drop_offset(const Drop& d) {
  if (d.dev_offset == nullptr) return make_uint2(d.off0, d.off1);
  const long long more = d.dev_bits == 64 ? *(const long long*)d.dev_offset : (long long)*(const int*)d.dev_offset;
  const unsigned long long o = (((unsigned long long)d.off1 << 32) | d.off0) + (unsigned long long)more;
  return make_uint2((uint32_t)o, (uint32_t)(o >> 32));
}

FO_DEVI uint4 philox(const Drop& d, const uint2 off, const uint32_t c0, const uint32_t c1) {
  uint32_t x0 = c0, x1 = c1, x2 = off.x, x3 = off.y;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)x0 * 0xD2511F53u, b = (unsigned long long)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ d.key[2 * r];
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ d.key[2 * r + 1];
    x3 = (uint32_t)a;
  }
  return make_uint4(x0, x1, x2, x3);
}

// The upper halves for the eight elements of a block, two to a word.  A tie, one element in 2^16, is settled here: its half becomes all ones where the
// element stays and zero where it does not, so that the eight need a shift and two comparisons per pair (`stays`).
FO_DEVI uint4 settle_ties(const Drop& d, const uint2 off, const uint32_t c0, const uint32_t c1, uint4 w) {
  const uint4 low = philox(d, off, c0, c1 | 0x80000000u);
  auto settle = [&](uint32_t& v, const uint32_t u) {
    if (((v ^ d.hi) & 0xFFFFu) == 0) v = (v & 0xFFFF0000u) | ((u & 0xFFFFu) >= d.lo ? 0xFFFFu : 0u);
    if ((v ^ d.hi) < 0x10000u) v = (v & 0xFFFFu) | ((u >> 16) >= d.lo ? 0xFFFF0000u : 0u);
  };
  settle(w.x, low.x);
  settle(w.y, low.y);
  settle(w.z, low.z);
  settle(w.w, low.w);
  return w;
}
FO_DEVI uint4 draw8(const Drop& d, const uint2 off, const unsigned long long block) {
  const uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);  // (below 2^61 blocks: the top bit is the second stream's)
  uint4 w = philox(d, off, c0, c1);
  if (d.lo != 0) {
    const uint32_t least = __vminu2(__vminu2(w.x ^ d.hi, w.y ^ d.hi), __vminu2(w.z ^ d.hi, w.w ^ d.hi));
    if ((least & 0xFFFFu) == 0 || least < 0x10000u) w = settle_ties(d, off, c0, c1, w);
  }
  return w;
}
FO_DEVI bool stays(const Drop& d, const uint4& w, const int j) {
  const uint32_t v = j < 2 ? w.x : (j < 4 ? w.y : (j < 6 ? w.z : w.w));
  return ((j & 1) != 0 ? v : v << 16) > d.above;
}
// Bit j: element 8 * block + j stays.
FO_DEVI uint32_t keep8(const Drop& d, const uint2 off, const unsigned long long block) {
  const uint4 w = draw8(d, off, block);
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) keep |= (stays(d, w, j) ? 1u : 0u) << j;
  return keep;
}

// ---- eight elements as fp32 ----------------------------------------------------------------------------------------
template <int DT>
struct Oct;  // as they lie in memory
template <>
struct Oct<FO_F32> {
  uint4 a, b;
  FO_DEVI void get(float (&v)[8]) const {
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
  }
  FO_DEVI void set(const float (&v)[8]) {
    a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  }
  FO_DEVI void load(const void* p) { a = ((const uint4*)p)[0]; b = ((const uint4*)p)[1]; }
  FO_DEVI void store(void* p) const { ((uint4*)p)[0] = a; ((uint4*)p)[1] = b; }
};
template <int DT>
struct Oct16 {
  uint4 a;
  FO_DEVI void get(float (&v)[8]) const {
    unpack2<DT>(a.x, v[0], v[1]); unpack2<DT>(a.y, v[2], v[3]); unpack2<DT>(a.z, v[4], v[5]); unpack2<DT>(a.w, v[6], v[7]);
  }
  FO_DEVI void set(const float (&v)[8]) { a = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])); }
  FO_DEVI void load(const void* p) { a = *(const uint4*)p; }
  FO_DEVI void store(void* p) const { *(uint4*)p = a; }
};
template <>
struct Oct<FO_BF16> : Oct16<FO_BF16> {};
template <>
struct Oct<FO_F16> : Oct16<FO_F16> {};

__host__ __device__ constexpr int size_of(int dt) { return dt == FO_F32 ? 4 : 2; }

// one element, and back; rounded to nearest
template <int DT>
FO_DEVI float load1(const void* p, const unsigned long long i) {
  if constexpr (DT == FO_F32) return ((const float*)p)[i];
  else return Lp<DT>::to_f32(((const unsigned short*)p)[i]);
}
template <int DT>
FO_DEVI void store1(void* p, const unsigned long long i, const float v) {
  if constexpr (DT == FO_F32) ((float*)p)[i] = v;
  else ((unsigned short*)p)[i] = (unsigned short)Lp<DT>::from_f32(v);
}

// id of token n; negative where it is no token
FO_DEVI long long id_at(const void* ids, const int bits, const unsigned long long n) {
  return bits == 64 ? ((const long long*)ids)[n] : (long long)((const int*)ids)[n];
}

__host__ __device__ inline bool on_16_bytes(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace fo
