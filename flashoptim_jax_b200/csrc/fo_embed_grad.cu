// Gradient of an embedding lookup:  dW[v, :] (+)= sum over the tokens n with ids[n] = v, in ascending n, of
// scale * keep / (1 - p) * dY[n, :], in fp32, rounded once.
//
// Three steps.  (1) The tokens are sorted by id, stably (so the order of every sum is fixed: same inputs, same bits, no atomics on
// values).  (2) The sorted tokens are cut into chunks of equal length whatever their ids, so that an id that half of all
// tokens carry costs no more than others: a warp adds up 256 columns of one chunk, writes the rows whose tokens lie all in the
// chunk, and leaves a partial sum of the row at either end that does not.  (3) The partial sums of a row are added up.
#include <cooperative_groups.h>

#include "fo_tokens.cuh"

namespace fo {

namespace cg = cooperative_groups;

constexpr int kSms = 148;

// ---- sizes and the workspace ----------------------------------------------------------------------------------------
constexpr int kTileCols = 256;     // columns of a warp: eight per lane
constexpr int kSumThreads = 256;
constexpr int kLeastChunk = 4;     // tokens
constexpr int kSumWarps = kSms * 32;  // wanted

struct GradPlan {
  bool several;  // the sort takes several launches
  uint32_t tiles, chunk, chunks;
  uint32_t blocks;  // of such a sort
  unsigned long long key[2], pos[2], hist, total, partial, bytes;  // offsets in the workspace
};

constexpr int kDigitMax = 9, kBinsMax = 1 << kDigitMax;
// The sort of one cluster: eight blocks, which hold all tokens in shared memory.
constexpr int kCluster = 8, kSortThreads = 1024, kSortRounds = 8;
constexpr unsigned long long kSortMost = (unsigned long long)kCluster * kSortThreads * kSortRounds;
constexpr int kSortRowBits = 27;  // of the rows, of which a bit each lies in the shared memory of the blocks beside it
// The sort over several launches: tiles of 4096 tokens.
constexpr int kRadixThreads = 512, kRadixRounds = 8, kRadixTile = kRadixThreads * kRadixRounds;

static GradPlan plan_of(const unsigned long long rows, const unsigned long long dim, const unsigned long long n) {
  GradPlan g = {};
  g.several = n > kSortMost || rows >> kSortRowBits != 0;
  g.tiles = (uint32_t)((dim + kTileCols - 1) / kTileCols);
  unsigned long long chunk = (n * g.tiles + kSumWarps - 1) / kSumWarps;
  if (chunk < kLeastChunk) chunk = kLeastChunk;
  if (chunk > n && n > 0) chunk = n;
  g.chunk = (uint32_t)chunk;
  g.chunks = (uint32_t)((n + chunk - 1) / chunk);
  g.blocks = (uint32_t)((n + kRadixTile - 1) / kRadixTile);
  unsigned long long at = 0;
  auto take = [&](unsigned long long bytes) {
    const unsigned long long here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int i = 0; i < (g.several ? 2 : 1); ++i) {
    g.key[i] = take(4 * n);
    g.pos[i] = take(4 * n);
  }
  if (g.several) {
    g.hist = take(4ull * kBinsMax * g.blocks);
    g.total = take(4ull * kBinsMax);
  }
  g.partial = take(8ull * g.chunks * g.tiles * kTileCols);
  g.bytes = at;
  return g;
}

// ---- (1) the sort ----------------------------------------------------------------------------------------------------
struct SortParams {
  const void* ids;
  uint32_t* key_out;
  uint32_t* pos_out;
  void* out;  // the gradient, whose rows without a token are cleared meanwhile; null: none are
  unsigned long long row_bytes;
  uint32_t n, rows, m;  // m: tokens of a block
  int32_t ids_bits, passes, digit_bits;
};

// Ids that name no row sort behind all rows.
FO_DEVI uint32_t key_of(const long long id, const uint32_t rows) { return id < 0 || id >= (long long)rows ? rows : (uint32_t)id; }

// Zeros from a to b (elements of 2 or 4 bytes) by one warp.
FO_DEVI void clear_bytes(char* a, char* const b, const int lane) {
  char* const up = (char*)(((uintptr_t)a + 15) & ~(uintptr_t)15);
  char* const down = (char*)((uintptr_t)b & ~(uintptr_t)15);
  if (up >= down) {
    for (char* c = a + 2 * lane; c < b; c += 64) *(unsigned short*)c = 0;
    return;
  }
  if (a + 2 * lane < up) *(unsigned short*)(a + 2 * lane) = 0;
  for (char* c = up + 16 * lane; c < down; c += 512) *(uint4*)c = make_uint4(0u, 0u, 0u, 0u);
  if (down + 2 * lane < b) *(unsigned short*)(down + 2 * lane) = 0;
}

// exclusive sum over the first kBinsMax threads of a block; all threads call it
FO_DEVI uint32_t scan_bins(const uint32_t v, uint32_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const uint32_t y = __shfl_up_sync(~0u, x, s);
    if (lane >= s) x += y;
  }
  if (lane == 31 && warp < kBinsMax / 32) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp && w < kBinsMax / 32; ++w) before += warp_sums[w];
  __syncthreads();
  return before + x - v;
}

// The place of a lane's token among those of its warp with the same digit so far; `counts`: the warp's, one per digit.  The lanes of one digit
// are found at once, the first of them counts for all.
FO_DEVI uint32_t rank_in_warp(const uint32_t digit, const bool valid, unsigned short* counts, const int lane) {
  const uint32_t same = __match_any_sync(~0u, valid ? digit : 0xFFFFFFFFu);
  uint32_t rank = 0;
  if (valid) rank = counts[digit] + __popc(same & ((1u << lane) - 1u));
  __syncwarp();
  if (valid && (same & ((1u << lane) - 1u)) == 0) counts[digit] += (unsigned short)__popc(same);
  __syncwarp();
  return rank;
}

struct SortShared {
  unsigned short counts[kSortThreads / 32][kBinsMax];
  uint32_t hist[2][kBinsMax];
  uint32_t base[kBinsMax];
  uint32_t warp_sums[kBinsMax / 32];
};

// Up to kSortMost tokens: one cluster sorts them, least digit first, its blocks' shared memory holding all keys and positions
// (a pass moves them through the cluster's shared memory, not through the L2, and its barriers are the hardware's), while the other
// blocks clear the rows of the gradient that no token names.
__global__ void __launch_bounds__(kSortThreads) __cluster_dims__(kCluster, 1, 1) sort_kernel(const __grid_constant__ SortParams p) {
  chain_wait();
  chain_release();
  extern __shared__ __align__(16) unsigned char sort_mem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= kCluster) {
    // this block's rows, a bit for each that a token names
    uint32_t* const named = (uint32_t*)sort_mem;
    const uint32_t f = blockIdx.x - kCluster, fs = gridDim.x - kCluster;
    const uint32_t first = (uint32_t)((unsigned long long)p.rows * f / fs), last = (uint32_t)((unsigned long long)p.rows * (f + 1) / fs);
    for (uint32_t i = threadIdx.x; i < (last - first + 31) / 32; i += kSortThreads) named[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.n; i += kSortThreads) {
      const uint32_t k = key_of(id_at(p.ids, p.ids_bits, i), p.rows);
      if (k >= first && k < last) atomicOr(&named[(k - first) / 32], 1u << ((k - first) & 31));
    }
    __syncthreads();
    for (uint32_t r = first + warp; r < last; r += kSortThreads / 32)
      if ((named[(r - first) / 32] >> ((r - first) & 31) & 1u) == 0) {
        char* const row = (char*)p.out + (unsigned long long)r * p.row_bytes;
        clear_bytes(row, row + p.row_bytes, lane);
      }
    return;
  }
  SortShared& s = *(SortShared*)sort_mem;
  uint2* const buffer[2] = {(uint2*)(sort_mem + sizeof(SortShared)), (uint2*)(sort_mem + sizeof(SortShared)) + p.m};
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t me = blockIdx.x, begin = me * p.m;
  const uint32_t mine = begin < p.n ? min(p.m, p.n - begin) : 0u;
  const uint32_t rounds = (p.m + kSortThreads - 1) / kSortThreads;
  const uint32_t at0 = warp * rounds * 32 + lane;  // a warp's tokens are neighbours, in rounds of 32
  const uint32_t bins = 1u << p.digit_bits;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit_bits;
    for (uint32_t i = threadIdx.x; i < sizeof(s.counts) / 4; i += kSortThreads) ((uint32_t*)s.counts)[i] = 0;
    __syncthreads();
    uint2 item[kSortRounds];
    uint32_t rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= (int)rounds) break;
      const uint32_t i = at0 + r * 32;
      const bool valid = i < mine;
      if (valid) item[r] = pass == 0 ? make_uint2(key_of(id_at(p.ids, p.ids_bits, begin + i), p.rows), begin + i) : buffer[(pass - 1) & 1][i];
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= (int)rounds) break;
      rank[r] = rank_in_warp((item[r].x >> shift) & (bins - 1), at0 + r * 32 < mine, s.counts[warp], lane);
    }
    __syncthreads();
    if (threadIdx.x < kBinsMax) {  // digit by digit: the warps' counts to places, and the block's count
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortThreads / 32; ++w) {
        const uint32_t c = s.counts[w][threadIdx.x];
        s.counts[w][threadIdx.x] = (unsigned short)sum;
        sum += c;
      }
      s.hist[pass & 1][threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t all = 0, before = 0;
    if (threadIdx.x < kBinsMax) {
      uint32_t h[kCluster];
#pragma unroll
      for (int b = 0; b < kCluster; ++b) h[b] = *cluster.map_shared_rank(&s.hist[pass & 1][threadIdx.x], b);
#pragma unroll
      for (int b = 0; b < kCluster; ++b) {
        if (b < (int)me) before += h[b];
        all += h[b];
      }
    }
    const uint32_t smaller = scan_bins(all, s.warp_sums);
    if (threadIdx.x < kBinsMax) s.base[threadIdx.x] = smaller + before;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= (int)rounds) break;
      if (at0 + r * 32 < mine) {
        const uint32_t digit = (item[r].x >> shift) & (bins - 1);
        const uint32_t to = s.base[digit] + s.counts[warp][digit] + rank[r];
        if (pass + 1 == p.passes) {
          p.key_out[to] = item[r].x;
          p.pos_out[to] = item[r].y;
        } else {
          const uint32_t b = to / p.m;
          cluster.map_shared_rank(buffer[pass & 1], b)[to - b * p.m] = item[r];
        }
      }
    }
    cluster.sync();  // also: no block ends while another reads its histogram
  }
}

// Clears the whole gradient; beside the first launch of a long sort.
struct RadixParams {
  const void* ids;
  const uint32_t* key_in;  // null: the ids
  const uint32_t* pos_in;
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* hist;   // [bin][block]
  uint32_t* total;  // [bin]
  void* out;
  unsigned long long out_bytes;
  uint32_t n, rows, blocks;
  int32_t ids_bits, shift, digit_bits;
};
FO_DEVI uint32_t radix_key(const RadixParams& p, const uint32_t i) { return p.key_in != nullptr ? p.key_in[i] : key_of(id_at(p.ids, p.ids_bits, i), p.rows); }

__global__ void __launch_bounds__(kRadixThreads) radix_count_kernel(const __grid_constant__ RadixParams p) {
  chain_wait();
  chain_release();
  if (blockIdx.x >= p.blocks) {
    const unsigned long long warps = (unsigned long long)(gridDim.x - p.blocks) * (kRadixThreads / 32), w = (unsigned long long)(blockIdx.x - p.blocks) * (kRadixThreads / 32) + threadIdx.x / 32;
    const unsigned long long step = 8192, pieces = (p.out_bytes + step - 1) / step;
    for (unsigned long long i = w; i < pieces; i += warps)
      clear_bytes((char*)p.out + i * step, (char*)p.out + (i + 1 < pieces ? (i + 1) * step : p.out_bytes), threadIdx.x & 31);
    return;
  }
  __shared__ uint32_t count[kBinsMax];
  for (int i = threadIdx.x; i < kBinsMax; i += kRadixThreads) count[i] = 0;
  __syncthreads();
  const uint32_t mask = (1u << p.digit_bits) - 1u;
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) {
    const unsigned long long i = (unsigned long long)blockIdx.x * kRadixTile + r * kRadixThreads + threadIdx.x;
    if (i < p.n) atomicAdd(&count[(radix_key(p, (uint32_t)i) >> p.shift) & mask], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBinsMax; i += kRadixThreads) p.hist[(unsigned long long)i * p.blocks + blockIdx.x] = count[i];
}

// Per digit: the blocks' counts to places, and the total.  One block per digit.
constexpr int kRadixScanThreads = 256;
__global__ void __launch_bounds__(kRadixScanThreads) radix_scan_kernel(const __grid_constant__ RadixParams p) {
  chain_wait();
  chain_release();
  __shared__ uint32_t sums[kRadixScanThreads / 32];
  uint32_t* const h = p.hist + (unsigned long long)blockIdx.x * p.blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (uint32_t b0 = 0; b0 < p.blocks; b0 += kRadixScanThreads) {
    const uint32_t b = b0 + threadIdx.x;
    const uint32_t v = b < p.blocks ? h[b] : 0u;
    uint32_t x = v;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t y = __shfl_up_sync(~0u, x, s);
      if (lane >= s) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    uint32_t before = carry;
    for (int w = 0; w < warp; ++w) before += sums[w];
    if (b < p.blocks) h[b] = before + x - v;
    for (int w = 0; w < kRadixScanThreads / 32; ++w) carry += sums[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.total[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kRadixThreads) radix_scatter_kernel(const __grid_constant__ RadixParams p) {
  chain_wait();
  chain_release();
  __shared__ unsigned short counts[kRadixThreads / 32][kBinsMax];
  __shared__ uint32_t base[kBinsMax];
  __shared__ uint32_t warp_sums[kBinsMax / 32];
  static_assert(kRadixThreads == kBinsMax, "a thread per digit");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t i = threadIdx.x; i < sizeof(counts) / 4; i += kRadixThreads) ((uint32_t*)counts)[i] = 0;
  __syncthreads();
  const uint32_t mask = (1u << p.digit_bits) - 1u;
  const unsigned long long i0 = (unsigned long long)blockIdx.x * kRadixTile + warp * (kRadixRounds * 32) + lane;
  uint32_t key[kRadixRounds], rank[kRadixRounds];
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) key[r] = i0 + r * 32 < p.n ? radix_key(p, (uint32_t)(i0 + r * 32)) : 0u;
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) rank[r] = rank_in_warp((key[r] >> p.shift) & mask, i0 + r * 32 < p.n, counts[warp], lane);
  __syncthreads();
  uint32_t sum = 0;
#pragma unroll 4
  for (int w = 0; w < kRadixThreads / 32; ++w) {
    const uint32_t c = counts[w][threadIdx.x];
    counts[w][threadIdx.x] = (unsigned short)sum;
    sum += c;
  }
  const uint32_t smaller = scan_bins(threadIdx.x <= mask ? p.total[threadIdx.x] : 0u, warp_sums);
  base[threadIdx.x] = smaller + p.hist[(unsigned long long)threadIdx.x * p.blocks + blockIdx.x];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) {
    if (i0 + r * 32 < p.n) {
      const uint32_t digit = (key[r] >> p.shift) & mask, to = base[digit] + counts[warp][digit] + rank[r];
      if (to >= p.n) continue;  // (ids that another stream changed meanwhile)
      p.key_out[to] = key[r];
      p.pos_out[to] = p.pos_in != nullptr ? p.pos_in[i0 + r * 32] : (uint32_t)(i0 + r * 32);
    }
  }
}

// ---- (2) and (3) the sums --------------------------------------------------------------------------------------------
struct SumParams {
  const void* dy;
  const uint32_t* key;
  const uint32_t* pos;
  void* out;
  float* partial;  // [chunk][first, last][tiles * kTileCols]
  unsigned long long n, dim, dy_stride;
  uint32_t rows, tiles, chunk, chunks;
  int32_t out_dtype, accumulate, out_vectors;
  float factor;
  Drop drop;
};

// Eight columns of a row of the gradient, from c on (`count` of them inside the row).
FO_DEVI void write_row(const SumParams& p, const uint32_t row, const unsigned long long c, const int count, float (&v)[8]) {
  const unsigned long long at = (unsigned long long)row * p.dim + c;
  auto go = [&](auto tag) {
    constexpr int DT = decltype(tag)::value;
    if (count == 8 && p.out_vectors) {
      char* const to = (char*)p.out + at * size_of(DT);
      Oct<DT> o;
      if (p.accumulate) {
        float old[8];
        o.load(to);
        o.get(old);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fadd(old[j], v[j]);
      }
      o.set(v);
      o.store(to);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < count) store1<DT>(p.out, at + j, p.accumulate ? fadd(load1<DT>(p.out, at + j), v[j]) : v[j]);
    }
  };
  if (p.out_dtype == FO_F32) go(std::integral_constant<int, FO_F32>{});
  else if (p.out_dtype == FO_BF16) go(std::integral_constant<int, FO_BF16>{});
  else go(std::integral_constant<int, FO_F16>{});
}

// Bound by HBM: every row of dY is read once, in pieces of 512 bytes (1 KB in fp32) wherever the sort has put it; kAhead of them are in flight per warp.
constexpr int kAhead = 4;
template <int DT, bool VECTORS>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const __grid_constant__ SumParams p) {
  chain_wait();
  chain_release();
  Drop d = p.drop;
  resolve_offset(d);
  const int lane = threadIdx.x & 31;
  const unsigned long long task = (unsigned long long)blockIdx.x * (kSumThreads / 32) + threadIdx.x / 32;
  if (task >= (unsigned long long)p.chunks * p.tiles) return;
  const uint32_t tile = (uint32_t)(task % p.tiles), chunk = (uint32_t)(task / p.tiles);
  const unsigned long long first = (unsigned long long)chunk * p.chunk, last = min(first + p.chunk, p.n);
  const unsigned long long c = (unsigned long long)tile * kTileCols + lane * 8;
  const int count = c >= p.dim ? 0 : (p.dim - c < 8 ? (int)(p.dim - c) : 8);
  const uint32_t behind = last < p.n ? p.key[last] : 0xFFFFFFFFu;
  uint32_t row = p.key[first];
  bool open = first > 0 && p.key[first - 1] == row;  // the row began in an earlier chunk
  float sum[8] = {};
  float* const partial = p.partial + ((unsigned long long)chunk * 2 * p.tiles + tile) * kTileCols + lane * 8;
  auto leave = [&](float* to) {
    ((float4*)to)[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    ((float4*)to)[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
  };
  for (unsigned long long i0 = first; i0 < last && row < p.rows; i0 += kAhead) {
    Oct<DT> x[kAhead];
    float one[VECTORS ? 1 : kAhead][8];
    uint32_t key[kAhead], pos[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      key[k] = i0 + k < last ? p.key[i0 + k] : 0xFFFFFFFFu;
      pos[k] = i0 + k < last ? p.pos[i0 + k] : 0u;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (key[k] >= p.rows) break;
      const unsigned long long at = (unsigned long long)pos[k] * p.dy_stride + c;
      if constexpr (VECTORS) {
        if (count > 0) x[k].load((const char*)p.dy + at * size_of(DT));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) one[k][j] = j < count ? load1<DT>(p.dy, at + j) : 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= last) break;
      if (key[k] != row) {  // (the same for the whole warp)
        if (open) leave(partial);
        else if (count > 0) write_row(p, row, c, count, sum);
        open = false;
        row = key[k];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
      }
      if (row >= p.rows) break;
      float v[8];
      if constexpr (VECTORS) {
        if (count > 0) x[k].get(v);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = one[k][j];
      }
      const uint32_t keep = d.on ? keep8_from(d, (unsigned long long)pos[k] * p.dim + c) : 0xFFu;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] = fadd(sum[j], (keep >> j & 1u) != 0 ? fmul(v[j], p.factor) : 0.0f);
    }
  }
  if (row >= p.rows) return;
  if (open) leave(partial);  // (a row that began before and goes on behind leaves this one alone)
  else if (behind == row) leave(partial + (unsigned long long)p.tiles * kTileCols);
  else if (count > 0) write_row(p, row, c, count, sum);
}

// The rows whose tokens lie in several chunks: a block per chunk that such a row begins in, and tile of columns; the partial sums are
// dealt out to the block's warps and added up in a fixed order.
__global__ void __launch_bounds__(kSumThreads) join_kernel(const __grid_constant__ SumParams p) {
  chain_wait();
  chain_release();
  constexpr int kWarps = kSumThreads / 32;
  __shared__ float part[kWarps][kTileCols];
  const uint32_t tile = blockIdx.x % p.tiles, chunk = blockIdx.x / p.tiles;
  const unsigned long long first = (unsigned long long)chunk * p.chunk, next = first + p.chunk;
  if (next >= p.n) return;
  const uint32_t row = p.key[next];
  if (row >= p.rows || p.key[next - 1] != row) return;            // no row goes on from this chunk
  if (p.key[first] == row && first > 0 && p.key[first - 1] == row) return;  // it began earlier
  // the first chunk behind it that does not begin with the row
  uint32_t lo = chunk + 1, hi = p.chunks;  // lo begins with it
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (p.key[(unsigned long long)mid * p.chunk] == row) lo = mid; else hi = mid;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long width = (unsigned long long)p.tiles * kTileCols;
  const float* const at = p.partial + (unsigned long long)tile * kTileCols + lane * 8;
  float sum[8] = {};
  auto add = [&](const float* from) {
    const float4 a = ((const float4*)from)[0], b = ((const float4*)from)[1];
    sum[0] = fadd(sum[0], a.x); sum[1] = fadd(sum[1], a.y); sum[2] = fadd(sum[2], a.z); sum[3] = fadd(sum[3], a.w);
    sum[4] = fadd(sum[4], b.x); sum[5] = fadd(sum[5], b.y); sum[6] = fadd(sum[6], b.z); sum[7] = fadd(sum[7], b.w);
  };
  if (warp == 0) add(at + ((unsigned long long)chunk * 2 + 1) * width);
#pragma unroll 4
  for (uint32_t k = chunk + 1 + warp; k <= lo; k += kWarps) add(at + (unsigned long long)k * 2 * width);
#pragma unroll
  for (int j = 0; j < 8; ++j) part[warp][lane * 8 + j] = sum[j];
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    for (int w = 1; w < kWarps; ++w) sum[j] = fadd(sum[j], part[w][lane * 8 + j]);
  const unsigned long long c = (unsigned long long)tile * kTileCols + lane * 8;
  const int count = c >= p.dim ? 0 : (p.dim - c < 8 ? (int)(p.dim - c) : 8);
  if (count > 0) write_row(p, row, c, count, sum);
}

static int sizes_ok(const char* who, uint64_t rows, uint64_t dim, uint64_t n) {
  if (rows >= 0x7FFFFFFFull || n >= 0x7FFFFFFFull || dim >> 24)
    return fail(FO_ERR_TOO_LARGE, "%s: %llu tokens, %llu rows of %llu elements", who, (unsigned long long)n, (unsigned long long)rows, (unsigned long long)dim);
  return FO_OK;
}

// The smallest number of passes of at most kDigitMax bits that sorts keys 0 ... rows.
static void digits(uint32_t rows, int& passes, int& bits) {
  int width = 1;
  while ((rows >> width) != 0) ++width;
  passes = (width + kDigitMax - 1) / kDigitMax;
  bits = (width + passes - 1) / passes;
}

constexpr int kSortSmem = 200 * 1024;
static_assert(sizeof(SortShared) + 2 * sizeof(uint2) * kSortThreads * kSortRounds <= kSortSmem && (1u << kSortRowBits) / ((kSms - kCluster) / kCluster * kCluster) / 8 + 64 <= kSortSmem, "shared memory of the sort");
static int sort_in_cluster(const FoEmbedGrad& f, const GradPlan& g, cudaStream_t stream) {
  SortParams p = {};
  char* const ws = (char*)f.workspace;
  p.ids = f.ids; p.ids_bits = f.ids_bits;
  p.key_out = (uint32_t*)(ws + g.key[0]); p.pos_out = (uint32_t*)(ws + g.pos[0]);
  p.n = (uint32_t)f.n_tokens; p.rows = (uint32_t)f.rows;
  p.m = (p.n + kCluster - 1) / kCluster;
  digits(p.rows, p.passes, p.digit_bits);
  p.out = f.accumulate ? nullptr : f.out;
  p.row_bytes = f.dim * size_of(f.out_dtype);
  unsigned int grid = kCluster;
  if (!f.accumulate) grid += (kSms - kCluster) / kCluster * kCluster;
  const size_t bits_bytes = (p.rows / (grid > kCluster ? grid - kCluster : 1) + 64) / 32 * 4;
  size_t smem = sizeof(SortShared) + 2 * sizeof(uint2) * (size_t)p.m;
  if (!f.accumulate && bits_bytes > smem) smem = bits_bytes;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(FO_ERR_CUDA, "fo_embed_grad: cannot query the current device");
  if (dev >= 64 || (ready.load() >> dev & 1) == 0) {
    if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) != cudaSuccess)
      return fail(FO_ERR_CUDA, "fo_embed_grad: cannot set the shared memory size");
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  bool chained = true;
  const cudaError_t e = launch_chained(sort_kernel, grid, (unsigned int)kSortThreads, (int)smem, chained, stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}

// The sort over several launches; key[passes & 1] holds the result.
static int sort_in_memory(const FoEmbedGrad& f, const GradPlan& g, cudaStream_t stream, int& result) {
  char* const ws = (char*)f.workspace;
  RadixParams p = {};
  int passes;
  digits((uint32_t)f.rows, passes, p.digit_bits);
  p.ids = f.ids; p.ids_bits = f.ids_bits;
  p.hist = (uint32_t*)(ws + g.hist); p.total = (uint32_t*)(ws + g.total);
  p.n = (uint32_t)f.n_tokens; p.rows = (uint32_t)f.rows; p.blocks = g.blocks;
  p.out = f.out; p.out_bytes = f.rows * f.dim * size_of(f.out_dtype);
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < passes && e == cudaSuccess; ++pass) {
    p.key_in = pass == 0 ? nullptr : (const uint32_t*)(ws + g.key[(pass - 1) & 1]);
    p.pos_in = pass == 0 ? nullptr : (const uint32_t*)(ws + g.pos[(pass - 1) & 1]);
    p.key_out = (uint32_t*)(ws + g.key[pass & 1]); p.pos_out = (uint32_t*)(ws + g.pos[pass & 1]);
    p.shift = pass * p.digit_bits;
    result = pass & 1;
    bool chained = true;
    const unsigned int clearing = pass == 0 && !f.accumulate ? 2 * kSms : 0;
    e = launch_chained(radix_count_kernel, p.blocks + clearing, (unsigned int)kRadixThreads, 0, chained, stream, p);
    if (e == cudaSuccess) e = launch_chained(radix_scan_kernel, 1u << p.digit_bits, (unsigned int)kRadixScanThreads, 0, chained, stream, p);
    if (e == cudaSuccess) e = launch_chained(radix_scatter_kernel, p.blocks, (unsigned int)kRadixThreads, 0, chained, stream, p);
  }
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}

}  // namespace fo

using namespace fo;

extern "C" int fo_embed_grad_workspace(uint64_t rows, uint64_t dim, uint64_t n_tokens, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad_workspace: null pointer");
  *bytes = 0;
  if (int rc = sizes_ok("fo_embed_grad_workspace", rows, dim, n_tokens)) return rc;
  if (rows != 0 && dim != 0) *bytes = plan_of(rows, dim, n_tokens).bytes;
  return FO_OK;
}

extern "C" int fo_embed_grad(const FoEmbedGrad* f, void* cuda_stream) {
  if (f == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: null descriptor");
  if (f->struct_size != sizeof(FoEmbedGrad)) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: struct_size %u != %zu (ABI mismatch)", f->struct_size, sizeof(FoEmbedGrad));
  if (f->dy_dtype < FO_F32 || f->dy_dtype > FO_F16) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: bad dy_dtype %d", f->dy_dtype);
  if (f->out_dtype < FO_F32 || f->out_dtype > FO_F16) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: bad out_dtype %d", f->out_dtype);
  if (f->ids_bits != 32 && f->ids_bits != 64) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: ids_bits %d (32 or 64)", f->ids_bits);
  SumParams p = {};
  double factor;
  if (!make_drop(&f->dropout, p.drop, factor)) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: p = %g (it lies in [0, 1]), dev_offset_bits = %d (32 or 64)", f->dropout.p, f->dropout.dev_offset_bits);
  if (int rc = sizes_ok("fo_embed_grad", f->rows, f->dim, f->n_tokens)) return rc;
  if (f->rows == 0 || f->dim == 0 || (f->accumulate && f->n_tokens == 0)) return FO_OK;
  if (f->out == nullptr || (f->n_tokens > 0 && (f->ids == nullptr || f->dy == nullptr))) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: null pointer");
  if (f->dy_stride < f->dim || f->dy_stride >> 28) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: rows %llu elements apart are %llu long", (unsigned long long)f->dy_stride, (unsigned long long)f->dim);
  const GradPlan g = plan_of(f->rows, f->dim, f->n_tokens);
  if (f->workspace_bytes < g.bytes || (g.bytes > 0 && (f->workspace == nullptr || !on_16_bytes(f->workspace))))
    return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: a workspace of %llu bytes, aligned to 16, is needed, got %llu", (unsigned long long)g.bytes, (unsigned long long)f->workspace_bytes);
  cudaStream_t stream = (cudaStream_t)cuda_stream;
  int at = 0;
  if (int rc = g.several ? sort_in_memory(*f, g, stream, at) : sort_in_cluster(*f, g, stream)) return rc;
  if (f->n_tokens == 0) return FO_OK;
  char* const ws = (char*)f->workspace;
  p.dy = f->dy; p.out = f->out;
  p.key = (const uint32_t*)(ws + g.key[at]); p.pos = (const uint32_t*)(ws + g.pos[at]);
  p.partial = (float*)(ws + g.partial);
  p.n = f->n_tokens; p.dim = f->dim; p.dy_stride = f->dy_stride;
  p.rows = (uint32_t)f->rows; p.tiles = g.tiles; p.chunk = g.chunk; p.chunks = g.chunks;
  p.out_dtype = f->out_dtype; p.accumulate = f->accumulate != 0;
  p.out_vectors = on_16_bytes(f->out) && f->dim * size_of(f->out_dtype) % 16 == 0;
  p.factor = (float)(f->scale * factor);
  const bool vectors = f->dim % 8 == 0 && on_16_bytes(f->dy) && f->dy_stride * size_of(f->dy_dtype) % 16 == 0;
  void (*kernel)(const SumParams) = nullptr;
#define X(D) \
  if (f->dy_dtype == D) kernel = vectors ? sum_kernel<D, true> : sum_kernel<D, false>;
  X(FO_F32) X(FO_BF16) X(FO_F16)
#undef X
  const unsigned long long tasks = (unsigned long long)g.chunks * g.tiles, blocks = (tasks + kSumThreads / 32 - 1) / (kSumThreads / 32);
  if (tasks > 0x7FFFFFFFull) return fail(FO_ERR_TOO_LARGE, "fo_embed_grad: %llu tokens of %llu elements exceed one launch", (unsigned long long)f->n_tokens, (unsigned long long)f->dim);
  bool chained = true;
  cudaError_t e = launch_chained(kernel, (unsigned int)blocks, (unsigned int)kSumThreads, 0, chained, stream, p);
  if (e == cudaSuccess) e = launch_chained(join_kernel, (unsigned int)tasks, (unsigned int)kSumThreads, 0, chained, stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}
