// Embedding lookup:  out[n, :] = drop(scale * W[ids[n], :]), W stored in fp32 or 16 bits, or split into a 16-bit
// parameter and its error-correction code (the rows are then the fp32 weights that reconstruct_leaf gives).
#include "fo_tokens.cuh"

namespace fo {

constexpr int kEmbedThreads = 128;

struct EmbedParams {
  const void* table;
  const void* ecc;
  const void* ids;
  void* out;
  unsigned long long n_tokens, rows, dim;
  unsigned long long row_stride, ecc_stride;  // elements
  uint32_t tiles;  // of 256 columns
  int32_t ids_bits, out_f32;
  float factor;  // scale, and 1 / (1 - p)
  Drop drop;
};

template <int ECC>
struct EccOct {
  uint4 a;
  FO_DEVI void load(const void* p) {
    if constexpr (ECC == 16) a = *(const uint4*)p;
    if constexpr (ECC == 8) { const uint2 b = *(const uint2*)p; a = make_uint4(b.x, b.y, 0u, 0u); }
  }
  FO_DEVI int get(const int j) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (ECC == 16) return (int)(short)(w[j / 2] >> (16 * (j & 1)));
    if constexpr (ECC == 8) return (int)(signed char)(w[j / 4] >> (8 * (j & 3)));
    return 0;
  }
};

// A negative id is no token: zeros.  An id behind the last row reads nothing: a row of NaN, seen in the loss.
FO_DEVI float without_row(const long long id) { return id < 0 ? 0.0f : __int_as_float(0x7FC00000); }

// Eight elements of a row per thread, OCTS of them a block's width apart: the ids, then the rows, then the results.  Bound by HBM: 16384 tokens of 4096 bf16
// columns out of 128256 rows 37 us (193 MB, 5.2 TB/s; with one oct a thread 69, two 40, eight 42); 8192 tokens of 768 columns with dropout 6.9, of which the draws
// are 1.8 and launch and two trips to memory most.
// dim is a multiple of 8, all rows start on 16 bytes (codes of 8 bits: on 8).  INDEX: 32 bits where dim / 8 * n_tokens fits them.
template <int DT, int ECC, typename INDEX, int OCTS>
__global__ void __launch_bounds__(kEmbedThreads) embed_kernel(const __grid_constant__ EmbedParams p) {
  chain_wait();
  chain_release();
  const Drop& d = p.drop;
  const uint2 off = drop_offset(d);
  const INDEX per_row = (INDEX)(p.dim / 8), octs = (INDEX)p.n_tokens * per_row;
  const INDEX q0 = (INDEX)blockIdx.x * (kEmbedThreads * OCTS) + threadIdx.x;
  Oct<DT> x[OCTS];
  EccOct<ECC> e[OCTS];
  long long id[OCTS];
  INDEX col[OCTS];
#pragma unroll
  for (int k = 0; k < OCTS; ++k) {
    const INDEX q = q0 + k * kEmbedThreads;
    if (q >= octs) break;
    const INDEX n = q / per_row;
    col[k] = q - n * per_row;
    id[k] = id_at(p.ids, p.ids_bits, n);
  }
#pragma unroll
  for (int k = 0; k < OCTS; ++k) {
    const INDEX q = q0 + k * kEmbedThreads;
    if (q >= octs) break;
    if (id[k] < 0 || (unsigned long long)id[k] >= p.rows) continue;
    x[k].load((const char*)p.table + ((unsigned long long)id[k] * p.row_stride + (unsigned long long)col[k] * 8) * size_of(DT));
    if constexpr (ECC != 0) e[k].load((const char*)p.ecc + ((unsigned long long)id[k] * p.ecc_stride + (unsigned long long)col[k] * 8) * (ECC / 8));
  }
  uint4 w[OCTS];  // drawn while the rows are on their way
  if (d.on) {
#pragma unroll
    for (int k = 0; k < OCTS; ++k) w[k] = draw8(d, off, q0 + k * kEmbedThreads);
  }
#pragma unroll
  for (int k = 0; k < OCTS; ++k) {
    const INDEX q = q0 + k * kEmbedThreads;
    if (q >= octs) break;
    float v[8];
    if (id[k] < 0 || (unsigned long long)id[k] >= p.rows) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = without_row(id[k]);
    } else if constexpr (ECC == 0) {
      x[k].get(v);
    } else {
      const uint32_t h[4] = {x[k].a.x, x[k].a.y, x[k].a.z, x[k].a.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fast::reconstruct<DT, ECC>((h[j / 2] >> (16 * (j & 1))) & 0xFFFFu, e[k].get(j));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmul(v[j], p.factor);
    if (d.on) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = stays(d, w[k], j) ? v[j] : 0.0f;
    }
    if (DT == FO_F32 || p.out_f32) {
      Oct<FO_F32> y;
      y.set(v);
      y.store((char*)p.out + (unsigned long long)q * 32);
    } else {
      Oct<DT> y;
      y.set(v);
      y.store((char*)p.out + (unsigned long long)q * 16);
    }
  }
}

// Any width, stride and alignment: a warp per 256 columns of a token, every 32nd of them to a lane, so that neighbours lie in neighbouring lanes.  The id and
// all addresses are the warp's, worked out once; each lane draws for eight neighbours and hands them on.  5003 tokens of 1777 columns, fp16 with 16-bit codes, to
// fp32: 12.8 us in a graph (57 MB); eight neighbouring results per thread, whatever rows they lie in, took 27.
template <int DT, int ECC, bool F32>
__global__ void __launch_bounds__(kEmbedThreads) embed_any_kernel(const __grid_constant__ EmbedParams p) {
  chain_wait();
  chain_release();
  const Drop& d = p.drop;
  const int lane = threadIdx.x & 31;
  const unsigned long long task = (unsigned long long)blockIdx.x * (kEmbedThreads / 32) + threadIdx.x / 32;
  const unsigned long long n = task / p.tiles;
  if (n >= p.n_tokens) return;
  const uint32_t c0 = (uint32_t)(task - n * p.tiles) * 256;
  const int count = (int)min(256u, (uint32_t)p.dim - c0) - lane;  // columns from the lane's first one on
  const long long id = id_at(p.ids, p.ids_bits, n);
  const bool named = id >= 0 && (unsigned long long)id < p.rows;
  const unsigned long long row = named ? (unsigned long long)id : 0ull;
  const char* const w = (const char*)p.table + (row * p.row_stride + c0 + lane) * size_of(DT);
  const char* const e = (const char*)p.ecc + (row * p.ecc_stride + c0 + lane) * (ECC / 8);
  float v[8];
  int code[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = without_row(id);
    if (named && j * 32 < count) {
      v[j] = __uint_as_float(DT == FO_F32 ? ((const uint32_t*)w)[j * 32] : ((const unsigned short*)w)[j * 32]);
      if constexpr (ECC == 16) code[j] = ((const short*)e)[j * 32];
      if constexpr (ECC == 8) code[j] = ((const signed char*)e)[j * 32];
    }
  }
  const unsigned long long e0 = n * p.dim + c0;
  uint32_t low = 0xFFu, high = 0xFFu;  // the warp's 256 columns lie in 32 or 33 blocks of eight
  if (d.on) {
    const uint2 off = drop_offset(d);
    low = keep8(d, off, (e0 >> 3) + lane);
    if ((e0 & 7) != 0) high = keep8(d, off, (e0 >> 3) + 32);
  }
  char* const to = (char*)p.out + (e0 + lane) * (F32 ? 4 : size_of(DT));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (named) {
      if constexpr (ECC != 0) v[j] = fast::reconstruct<DT, ECC>(__float_as_uint(v[j]), code[j]);
      else if constexpr (DT != FO_F32) v[j] = Lp<DT>::to_f32(__float_as_uint(v[j]));
    }
    v[j] = fmul(v[j], p.factor);
    if (d.on) {
      const uint32_t at = ((uint32_t)e0 & 7u) + j * 32 + lane;
      const uint32_t bits = __shfl_sync(~0u, low, (at >> 3) & 31);
      if (((at >= 256 ? high : bits) >> (at & 7) & 1u) == 0) v[j] = 0.0f;
    }
    if (j * 32 < count) store1<F32 ? FO_F32 : DT>(to, j * 32, v[j]);
  }
}

template <int DT, int ECC>
static int launch_embed(const EmbedParams& p, const bool vectors, cudaStream_t stream) {
  const unsigned long long octs = p.n_tokens * (p.dim / 8), warps = p.n_tokens * p.tiles;
  constexpr int kOcts = 4;
  const unsigned long long per_block = vectors ? kEmbedThreads * kOcts : kEmbedThreads / 32, blocks = ((vectors ? octs : warps) + per_block - 1) / per_block;
  if (blocks > 0x7FFFFFFFull) return fail(FO_ERR_TOO_LARGE, "fo_embed: %llu tokens of %llu elements exceed one launch", p.n_tokens, p.dim);
  void (*kernel)(const EmbedParams) = p.out_f32 ? embed_any_kernel<DT, ECC, true> : embed_any_kernel<DT, ECC, DT == FO_F32>;
  if (vectors) kernel = octs < 0xFFFF0000ull ? embed_kernel<DT, ECC, uint32_t, kOcts> : embed_kernel<DT, ECC, unsigned long long, kOcts>;
  bool chained = true;
  const cudaError_t e = launch_chained(kernel, (unsigned int)blocks, (unsigned int)kEmbedThreads, 0, chained, stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed: launch failed: %s", cudaGetErrorString(e));
}

}  // namespace fo

using namespace fo;

extern "C" int fo_embed(const FoEmbed* f, void* stream) {
  if (f == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_embed: null descriptor");
  if (f->struct_size != sizeof(FoEmbed)) return fail(FO_ERR_INVALID_ARG, "fo_embed: struct_size %u != %zu (ABI mismatch)", f->struct_size, sizeof(FoEmbed));
  if (f->table_dtype < FO_F32 || f->table_dtype > FO_F16) return fail(FO_ERR_INVALID_ARG, "fo_embed: bad table_dtype %d", f->table_dtype);
  if (f->out_dtype != FO_F32 && f->out_dtype != f->table_dtype) return fail(FO_ERR_INVALID_ARG, "fo_embed: out_dtype %d (the table's or fp32)", f->out_dtype);
  if (f->ecc_bits != 0 && f->ecc_bits != 8 && f->ecc_bits != 16) return fail(FO_ERR_INVALID_ARG, "fo_embed: ecc_bits %d", f->ecc_bits);
  if (f->ecc_bits != 0 && f->table_dtype == FO_F32) return fail(FO_ERR_INVALID_ARG, "fo_embed: an fp32 table carries no ECC");
  if (f->ids_bits != 32 && f->ids_bits != 64) return fail(FO_ERR_INVALID_ARG, "fo_embed: ids_bits %d (32 or 64)", f->ids_bits);
  EmbedParams p;
  double factor;
  if (!make_drop(&f->dropout, p.drop, factor)) return fail(FO_ERR_INVALID_ARG, "fo_embed: p = %g (it lies in [0, 1]), dev_offset_bits = %d (32 or 64)", f->dropout.p, f->dropout.dev_offset_bits);
  if (!make_factor(f->scale, factor, p.factor)) return fail(FO_ERR_INVALID_ARG, "fo_embed: scale %g with p = %g (scale / (1 - p) has to be 0 or a normal fp32 number)", f->scale, f->dropout.p);
  if (f->n_tokens == 0 || f->dim == 0) return FO_OK;
  if (f->ids == nullptr || f->out == nullptr || (f->rows > 0 && (f->table == nullptr || (f->ecc_bits != 0 && f->ecc == nullptr))))
    return fail(FO_ERR_INVALID_ARG, "fo_embed: null pointer");
  if (f->row_stride < f->dim || (f->ecc_bits != 0 && f->ecc_stride < f->dim)) return fail(FO_ERR_INVALID_ARG, "fo_embed: rows %llu elements apart are %llu long", (unsigned long long)f->row_stride, (unsigned long long)f->dim);
  // element numbers, and byte addresses in the table, stay below 2^60
  if (f->n_tokens >> 32 || f->dim >> 28 || f->rows >> 32 || f->row_stride >> 28 || f->ecc_stride >> 28)
    return fail(FO_ERR_TOO_LARGE, "fo_embed: %llu tokens, %llu rows of %llu elements", (unsigned long long)f->n_tokens, (unsigned long long)f->rows, (unsigned long long)f->dim);
  p.table = f->table; p.ecc = f->ecc; p.ids = f->ids; p.out = f->out;
  p.n_tokens = f->n_tokens; p.rows = f->rows; p.dim = f->dim;
  p.row_stride = f->row_stride; p.ecc_stride = f->ecc_stride;
  p.tiles = (uint32_t)((p.dim + 255) / 256);
  p.ids_bits = f->ids_bits;
  p.out_f32 = f->out_dtype == FO_F32;
  const int size = size_of(f->table_dtype), code = f->ecc_bits / 8;
  const bool vectors = f->dim % 8 == 0 && on_16_bytes(f->table) && f->row_stride * size % 16 == 0 && on_16_bytes(f->out) &&
                       (code == 0 || ((uintptr_t)f->ecc % (8 * code) == 0 && f->ecc_stride % 8 == 0));
#define X(D, E) \
  if (f->table_dtype == D && f->ecc_bits == E) return launch_embed<D, E>(p, vectors, (cudaStream_t)stream);
  X(FO_F32, 0) X(FO_BF16, 0) X(FO_BF16, 8) X(FO_BF16, 16) X(FO_F16, 0) X(FO_F16, 8) X(FO_F16, 16)
#undef X
  return fail(FO_ERR_INVALID_ARG, "fo_embed: table_dtype %d with ecc_bits %d", f->table_dtype, f->ecc_bits);
}
