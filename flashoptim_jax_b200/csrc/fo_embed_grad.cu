// Gradient of an embedding lookup:  dW[v, :] (+)= sum over the tokens n with ids[n] = v, in ascending n, of
// scale * keep / (1 - p) * dY[n, :], in fp32, rounded once.
//
// Up to 64 tokens: one launch (few_kernel).  More: (1) the tokens are sorted by id, stably (so the order of every sum is fixed: same inputs, same bits, no
// atomics on values), which also says where each row's tokens begin.  (2) The sorted tokens are cut into chunks of equal length whatever their ids, so
// that an id that half of all tokens carry costs no more than others: a warp adds up 256 columns of one chunk and writes the rows whose tokens
// lie all in the chunk; of the row at either end that does not, it leaves a partial sum, and the warp that leaves a row's last one adds them
// up.  (3) The rows without a token are cleared in the launch of (2), mostly by blocks behind those of the sums.  (A launch of its own that starts beside the sums would read
// what the sort wrote without having waited for it: only a launch's own wait makes earlier ones' writes visible to it.)
//
// Bound by HBM from a hundred thousand rows of some thousand columns on (32768 tokens of 4096 bf16 columns into 128256 rows: 1.32 GB in 204 us, 6.5 TB/s), by
// latency below: the sort takes 5 to 11 us (three to six dependent trips to memory a launch), a chunk's sum as much, joining the pieces of
// frequent rows 3 to 5.  16384 tokens of 768 columns into 50257 rows, 102 MB: 31 us, 34 with dropout; 8192 tokens of 4096 columns added to what 128256
// rows hold: 39; 33 tokens: 7.5.  (Times in this file: whole calls in a graph, three sets of inputs in turn.)
#include "fo_tokens.cuh"

namespace fo {

constexpr int kSms = 148;

// ---- sizes and the workspace ----------------------------------------------------------------------------------------
constexpr int kTileCols = 256;     // columns of a warp: eight per lane
constexpr int kSumThreads = 256;
// Resident blocks per SM; about as many warps are wanted as are resident.  With dropout the registers of a third block are worth more to the draws (60000 tokens
// of 1024 columns into 50257 rows 80 us, 89 with three; without it 61 with two and 59 with three).
constexpr int sum_blocks_per_sm(const bool drop) { return drop ? 2 : 3; }
constexpr int kLeastChunk = 2;     // tokens
constexpr uint32_t kFewTokens = 64;  // up to so many take one launch and no workspace

// The sort by rows: 128 blocks, a 16-bit counter per row and warp; in one launch up to kSortAlone tokens, else in two, whatever
// the rows: the two ways meet near 8192 tokens (4096 tokens into 2999 rows 19.8 us in one launch and 23.0 in two, 2048 added to 128256 15.6 and 17.9; 8191 into 2999 29.3 and 29.6, 8192 into 50257
// 28.5 and 28.4, added to 128256 38.8 and 37.6, to 262143 20.0 and 20.6; 16384 into 50257 36.3 and 31.3).
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSortRows = 2048;                      // of a block, at most
constexpr uint32_t kSortBlocks = 128;
constexpr unsigned long long kSortMost = 65536;      // tokens
constexpr unsigned long long kSortAlone = 8192;  // of which up to so many take one launch
constexpr int kSortSmem = 220 * 1024;
static_assert(kSortRows == 2 * kSortThreads && (kSortWarps * 2 + 4) * (kSortRows + 2) + 4 * kSortAlone <= kSortSmem && kSortMost <= 65536 && kSortAlone % kSortThreads == 0,
              "two rows a thread, counters and lists in shared memory, places that fit the counters");
// More than 65536 tokens (a place no longer fits 16 bits) or 262143 rows (nor do the counters the shared memory): the sort by digits, three launches for each
// digit of at most nine bits, tiles of 4096 tokens.  It takes as long whatever the ids are: 131072 tokens of 768 columns into 50257 rows 97 us, 96 with 0.4 of the tokens of one id, where
// a sort by rows with counters of 32 bits took 13 less, and 41 more with that id, whose tokens are all one block's.
constexpr int kDigitMax = 9, kBinsMax = 1 << kDigitMax;
constexpr int kRadixThreads = 512, kRadixRounds = 8, kRadixTile = kRadixThreads * kRadixRounds;

struct GradPlan {
  bool alone, several;  // the sort takes one launch, or several per digit; otherwise two
  uint32_t tiles, chunk, chunks;
  uint32_t blocks;  // of a sort by digits
  unsigned int sort_smem;
  unsigned long long key[2], pos[2], starts, counters, hist, total, partial, bytes;  // offsets in the workspace
};

// (with dropout there are fewer chunks: the workspace without it has room for them)
static GradPlan plan_of(const unsigned long long rows, const unsigned long long dim, const unsigned long long n, const bool drop) {
  GradPlan g = {};
  if (n <= kFewTokens) {
    g.tiles = (uint32_t)((dim + kTileCols - 1) / kTileCols);
    return g;
  }
  g.several = n > kSortMost || rows >= (unsigned long long)kSortBlocks * kSortRows;
  const unsigned long long width = (rows / kSortBlocks + 2) & ~1ull, lists = 4 * ((n + kSortThreads - 1) / kSortThreads * kSortThreads);
  g.alone = !g.several && n <= kSortAlone;
  g.sort_smem = g.several ? 0u : (unsigned int)((kSortWarps * 2 + 4) * width + (g.alone ? lists : 0));
  g.tiles = (uint32_t)((dim + kTileCols - 1) / kTileCols);
  const unsigned long long warps = kSms * sum_blocks_per_sm(drop) * kSumThreads / 32;
  unsigned long long chunk = (n * g.tiles + warps - 1) / warps;
  if (chunk < kLeastChunk) chunk = kLeastChunk;
  if (chunk > n) chunk = n;
  g.chunk = (uint32_t)chunk;
  g.chunks = (uint32_t)((n + chunk - 1) / chunk);
  g.blocks = (uint32_t)((n + kRadixTile - 1) / kRadixTile);
  unsigned long long at = 0;
  auto take = [&](unsigned long long bytes) {
    const unsigned long long here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const unsigned long long dealt = (n + 2 * kSortThreads - 1) / (2 * kSortThreads) * (2 * kSortThreads);
  for (int i = 0; i < (g.alone ? 1 : 2); ++i) {
    g.key[i] = take(4 * dealt);
    g.pos[i] = take(4 * dealt);
  }
  g.starts = take(4 * (rows + 1));
  g.counters = take(12ull * g.chunks * g.tiles);
  if (!g.several && !g.alone) g.hist = take(4ull * kSortBlocks * (kSortMost / (2 * kSortThreads)));
  if (g.several) {
    g.hist = take(4ull * kBinsMax * g.blocks);
    g.total = take(4ull * kBinsMax);
  }
  g.partial = take(8ull * g.chunks * g.tiles * kTileCols);
  g.bytes = at;
  return g;
}

// ---- (1) the sort ----------------------------------------------------------------------------------------------------
// Ids that name no row sort behind all rows.
FO_DEVI uint32_t key_of(const long long id, const uint32_t rows) { return (unsigned long long)id < rows ? (uint32_t)id : rows; }

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

// The rows of up to 32 neighbours whose bits are set in `empty`, by one warp: row after row where a row keeps it busy, else in one go over the bytes of all.
constexpr uint32_t kLongRow = 512;  // bytes
FO_DEVI void clear_rows(char* const base, const uint32_t rows, const uint32_t empty, const unsigned long long row_bytes, const int lane) {
  if (row_bytes >= kLongRow) {
    for (uint32_t left = empty; left != 0; left &= left - 1u) {
      char* const row = base + (unsigned long long)(__ffs(left) - 1) * row_bytes;
      clear_bytes(row, row + row_bytes, lane);
    }
    return;
  }
  if (empty == 0) return;
  const int size = (int)row_bytes, total = (int)rows * size;
  for (int at = lane * 16 - (int)((uintptr_t)base & 15); at < total; at += 512) {
    if (at >= 0 && at + 16 <= total) {
      const uint32_t r0 = (uint32_t)at / size, r1 = (uint32_t)(at + 15) / size, mask = ((2u << r1) - 1u) & ~((1u << r0) - 1u);
      if ((empty & mask) == mask) {
        *(uint4*)(base + at) = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      if ((empty & mask) == 0) continue;
    }
    for (int b = max(at, 0); b < min(at + 16, total); b += 2)
      if ((empty >> ((uint32_t)b / size) & 1u) != 0) *(unsigned short*)(base + b) = 0;
  }
}

// Exclusive sum over the threads of a block of at most 1024; all of them call it.
FO_DEVI uint32_t scan_block(const uint32_t v, uint32_t* warp_sums, uint32_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const uint32_t y = __shfl_up_sync(~0u, x, s);
    if (lane >= s) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t sum = lane < warps ? warp_sums[lane] : 0u, before = lane < warp ? sum : 0u;
  sum = __reduce_add_sync(~0u, sum);
  before = __reduce_add_sync(~0u, before);
  __syncthreads();
  all = sum;
  return before + x - v;
}

// The place of a lane's token among those of its warp with the same digit so far; `counts`: the warp's, one per digit.  The lanes of one digit
// find one another bit by bit, where there are several digits among them; the first of them counts for all.
FO_DEVI uint32_t rank_in_warp(const uint32_t digit, const bool valid, const int bits, unsigned short* counts, const int lane) {
  uint32_t same = __ballot_sync(~0u, valid);
  const uint32_t one_of_them = __shfl_sync(~0u, digit, __ffs(same) - 1);
  if (__any_sync(~0u, valid && digit != one_of_them))
#pragma unroll 1
    for (int b = 0; b < bits; ++b) {
      const bool one = (digit >> b & 1u) != 0;
      const uint32_t ones = __ballot_sync(~0u, one);
      same &= one ? ones : ~ones;
    }
  const uint32_t before = __popc(same & ((1u << lane) - 1u));
  uint32_t rank = 0;
  if (valid) rank = counts[digit] + before;
  __syncwarp();
  if (valid && before == 0) counts[digit] = (unsigned short)(rank + __popc(same));
  __syncwarp();
  return rank;
}

struct SortParams {
  const void* ids;
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* starts;  // [rows + 1]: where the tokens of each row begin, in the order of slot_of
  uint32_t* counters;
  uint32_t n, rows, n_counters;
  int32_t ids_bits, row_bits;  // of a row's number within a block
};

// The order in which the sort by rows puts them: those of a block behind one another, block after block, row r belonging to block r % kSortBlocks.
// (Frequent ids are neighbours in most vocabularies: where ids come as 1 / rank, the first 1 / 128 of 50257 rows has half of all tokens, and its block took 30 us
// for 16384.)
__host__ __device__ inline uint32_t rows_before(const uint32_t block, const uint32_t rows) { return block * (rows / kSortBlocks) + min(block, rows % kSortBlocks); }
FO_DEVI uint32_t slot_of(const uint32_t row, const uint32_t rows) { return rows_before(row % kSortBlocks, rows) + row / kSortBlocks; }

// Up to kSortAlone tokens, in one launch and without a word between its blocks: each block has 1 / 128 of the rows.  It reads all ids (from the L2: at 64
// bytes a clock 16384 of them take 1 us), counts those of blocks in front of it, which is where its tokens begin in the order, and
// those of each of its rows, warp by warp, each warp having the tokens behind those of the one before and keeping a list of the block's among them; then
// each warp puts its list in place.  Eight blocks that sorted by digits through the shared memory of a cluster took 12.4 us for 8192 tokens, mostly waiting
// for one another.  Loops stay loops: unrolled, their code took longer to fetch than to run.
constexpr int kHitBits = 10;  // of a token's number within its warp's, and of its rank there: 32 warps x 2^10 = 32768 tokens
static_assert(kSortAlone <= (unsigned long long)kSortWarps << kHitBits && kSortRows <= 1 << (32 - 2 * kHitBits), "a hit is one word");
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const __grid_constant__ SortParams p) {
  chain_wait();
  chain_release();
  extern __shared__ __align__(16) unsigned char sort_mem[];
  __shared__ uint32_t warp_sums[kSortWarps];
  unsigned short* const counts = (unsigned short*)sort_mem;  // [warp][row]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t me = blockIdx.x, slots = rows_before(me, p.rows), mine = rows_before(me + 1, p.rows) - slots;
  const uint32_t width = (p.rows / kSortBlocks + 2) & ~1u;  // of a warp's counters
  uint32_t* const first = (uint32_t*)(sort_mem + (size_t)kSortWarps * width * 2);  // [row]
  const uint32_t rounds = (p.n + kSortThreads - 1) / kSortThreads;
  uint32_t* const list = first + width + warp * rounds * 32;  // row << 20 | rank among the warp's tokens of the row << 10 | token
  for (uint32_t i = threadIdx.x; i < kSortWarps * width / 2; i += kSortThreads) ((uint32_t*)counts)[i] = 0;
  for (uint32_t i = me * kSortThreads + threadIdx.x; i < p.n_counters; i += gridDim.x * kSortThreads) p.counters[i] = 0;
  const uint32_t i0 = warp * rounds * 32 + lane;
  unsigned short* const my_counts = counts + warp * width;
  constexpr int kAtOnce = 4;
  uint32_t below = 0, hits = 0;
  __syncthreads();
#pragma unroll 1
  for (uint32_t r0 = 0; r0 < rounds; r0 += kAtOnce) {
    uint32_t key[kAtOnce];
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) {
      const uint32_t i = i0 + (r0 + r) * 32;
      key[r] = r0 + r < rounds && i < p.n ? key_of(id_at(p.ids, p.ids_bits, i), p.rows) : p.rows;
    }
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) {
      const uint32_t block = key[r] < p.rows ? key[r] % kSortBlocks : kSortBlocks;
      below += block < me ? 1u : 0u;
      const bool in = block == me;
      const uint32_t found = __ballot_sync(~0u, in);
      if (found == 0) continue;
      const uint32_t rank = rank_in_warp(key[r] / kSortBlocks, in, p.row_bits, my_counts, lane);
      if (in) list[hits + __popc(found & ((1u << lane) - 1u))] = key[r] / kSortBlocks << 2 * kHitBits | rank << kHitBits | ((r0 + r) * 32 + lane);
      hits += __popc(found);
    }
  }
  uint32_t before, all;
  scan_block(below, warp_sums, before);
  // Per row: the warps' counts to places within the row, and its tokens; two rows a thread, neighbours.
  uint32_t total[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t row = threadIdx.x * 2 + j;
    if (row < mine) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = counts[w * width + row];
        counts[w * width + row] = (unsigned short)total[j];
        total[j] += c;
      }
    }
  }
  const uint32_t at = before + scan_block(total[0] + total[1], warp_sums, all);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t row = threadIdx.x * 2 + j;
    if (row < mine) p.starts[slots + row] = first[row] = j == 0 ? at : at + total[0];
  }
  if (me == kSortBlocks - 1 && threadIdx.x == 0) p.starts[p.rows] = before + all;
  __syncthreads();
  for (uint32_t h = lane; h < hits; h += 32) {
    const uint32_t hit = list[h], row = hit >> 2 * kHitBits;
    const uint32_t to = first[row] + my_counts[row] + (hit >> kHitBits & ((1u << kHitBits) - 1u));
    p.key_out[to] = row * kSortBlocks + me;
    p.pos_out[to] = warp * rounds * 32 + (hit & ((1u << kHitBits) - 1u));
  }
}

// More tokens than kSortAlone: two launches.  In the first, each block deals its 2048 tokens out to 128 piles by id % 128, each pile in the order of the
// tokens; in the second, block b takes the b-th piles of all, block after block, and puts their tokens in the order of the rows.  The work does not grow
// with blocks x tokens as above, where the sort of 32768 tokens took 29 us.  Bound by latency: about 11 us for 16384 tokens, beside one another, of which the loads and the
// barriers between them are most.
constexpr int kDealTokens = 2 * kSortThreads;
constexpr uint32_t kDealBlocksMost = kSortMost / kDealTokens;
struct DealParams {
  const void* ids;
  uint32_t* pile_key;  // [block][kDealTokens]
  uint32_t* pile_pos;
  uint32_t* pile_size;  // [block][kSortBlocks]
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* starts;
  uint32_t* counters;
  uint32_t n, rows, blocks, n_counters;
  int32_t ids_bits, row_bits;
};
__global__ void __launch_bounds__(kSortThreads) deal_kernel(const __grid_constant__ DealParams p) {
  chain_wait();
  chain_release();
  __shared__ unsigned short counts[kSortWarps][kSortBlocks];
  __shared__ uint32_t warp_sums[kSortWarps], first[kSortBlocks];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t key[2], rank[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint32_t i = blockIdx.x * kDealTokens + warp * 64 + r * 32 + lane;
    key[r] = i < p.n ? key_of(id_at(p.ids, p.ids_bits, i), p.rows) : p.rows;
  }
  for (uint32_t i = threadIdx.x; i < kSortWarps * kSortBlocks / 2; i += kSortThreads) ((uint32_t*)counts)[i] = 0;
  for (uint32_t i = blockIdx.x * kSortThreads + threadIdx.x; i < p.n_counters; i += gridDim.x * kSortThreads) p.counters[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r) rank[r] = rank_in_warp(key[r] % kSortBlocks, key[r] < p.rows, 7, counts[warp], lane);
  __syncthreads();
  uint32_t size = 0, all;
  if (threadIdx.x < kSortBlocks) {
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = (unsigned short)size;
      size += c;
    }
    p.pile_size[blockIdx.x * kSortBlocks + threadIdx.x] = size;
  }
  const uint32_t at = scan_block(size, warp_sums, all);
  if (threadIdx.x < kSortBlocks) first[threadIdx.x] = at;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (key[r] < p.rows) {
      const uint32_t pile = key[r] % kSortBlocks, to = blockIdx.x * kDealTokens + first[pile] + counts[warp][pile] + rank[r];
      p.pile_key[to] = key[r];
      p.pile_pos[to] = blockIdx.x * kDealTokens + warp * 64 + r * 32 + lane;
    }
}
__global__ void __launch_bounds__(kSortThreads) order_kernel(const __grid_constant__ DealParams p) {
  chain_wait();
  chain_release();
  extern __shared__ __align__(16) unsigned char sort_mem[];
  __shared__ uint32_t warp_sums[kSortWarps], pile_at[kDealBlocksMost], pile_begin[kDealBlocksMost + 1], smaller;
  unsigned short* const counts = (unsigned short*)sort_mem;  // [warp][row]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t me = blockIdx.x, slots = rows_before(me, p.rows), mine = rows_before(me + 1, p.rows) - slots;
  const uint32_t width = (p.rows / kSortBlocks + 2) & ~1u;
  uint32_t* const first = (uint32_t*)(sort_mem + (size_t)kSortWarps * width * 2);  // [row]
  // Where each block's pile begins and how large it is: a warp per block that dealt.
  static_assert(kDealBlocksMost <= kSortWarps && kSortBlocks == 128, "a warp per block, four piles a lane");
  if (warp < (int)p.blocks) {
    const uint4 c = ((const uint4*)(p.pile_size + warp * kSortBlocks))[lane];
    uint32_t before = 0;
    before += lane * 4 < me ? c.x : 0u;
    before += lane * 4 + 1 < me ? c.y : 0u;
    before += lane * 4 + 2 < me ? c.z : 0u;
    before += lane * 4 + 3 < me ? c.w : 0u;
    before = __reduce_add_sync(~0u, before);
    if (lane == (int)(me / 4)) {
      pile_at[warp] = warp * kDealTokens + before;
      pile_begin[warp + 1] = me % 4 == 0 ? c.x : (me % 4 == 1 ? c.y : (me % 4 == 2 ? c.z : c.w));
    }
    if (lane == 0) warp_sums[warp] = before;
  }
  for (uint32_t i = threadIdx.x; i < kSortWarps * width / 2; i += kSortThreads) ((uint32_t*)counts)[i] = 0;
  __syncthreads();
  if (warp == 0) {
    uint32_t x = lane < (int)p.blocks ? pile_begin[lane + 1] : 0u;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t y = __shfl_up_sync(~0u, x, s);
      if (lane >= s) x += y;
    }
    if (lane < (int)kDealBlocksMost) pile_begin[lane + 1] = x;
    if (lane == 0) pile_begin[0] = 0;
    const uint32_t sum = __reduce_add_sync(~0u, lane < (int)p.blocks ? warp_sums[lane] : 0u);
    if (lane == 0) smaller = sum;
  }
  __syncthreads();
  const uint32_t tokens = pile_begin[p.blocks], before = smaller;
  const uint32_t rounds = (tokens + kSortThreads - 1) / kSortThreads, warps = rounds == 0 ? 0u : (tokens + rounds * 32 - 1) / (rounds * 32);
  unsigned short* const my_counts = counts + warp * width;
  // f(key, rank among the warp's tokens of its row, position) for this block's tokens, four rounds' loads at once
  auto walk = [&](auto with_pos, auto f) {
    uint32_t pile = 0;  // the one that holds the lane's next token: sought once, then followed
    for (uint32_t step = kDealBlocksMost / 2; step != 0; step /= 2)
      if (pile + step < p.blocks && pile_begin[pile + step] <= warp * rounds * 32 + lane) pile += step;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < rounds; r0 += 4) {
      uint32_t key[4], pos[4];
      bool in[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t i = (warp * rounds + r0 + r) * 32 + lane;
        in[r] = r0 + r < rounds && i < tokens;
        while (pile + 1 < p.blocks && pile_begin[pile + 1] <= i) ++pile;
        const uint32_t from = pile_at[pile] + i - pile_begin[pile];
        key[r] = in[r] ? p.pile_key[from] : 0u;
        pos[r] = decltype(with_pos)::value && in[r] ? p.pile_pos[from] : 0u;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r0 + r >= rounds) break;
        const uint32_t rank = rank_in_warp(key[r] / kSortBlocks, in[r], p.row_bits, my_counts, lane);
        if (in[r]) f(key[r], rank, pos[r]);
      }
    }
  };
  uint32_t only_key = 0, only_rank = ~0u, only_pos = 0;  // of one round, which is the usual case, nothing is looked up again
  if (warp < (int)warps) {
    if (rounds == 1)
      walk(std::true_type{}, [&](const uint32_t key, const uint32_t rank, const uint32_t pos) { only_key = key, only_rank = rank, only_pos = pos; });
    else
      walk(std::false_type{}, [](uint32_t, uint32_t, uint32_t) {});
  }
  __syncthreads();
  uint32_t total[2] = {0u, 0u}, all;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t row = threadIdx.x * 2 + j;
    if (row < mine) {
#pragma unroll 4
      for (uint32_t w = 0; w < warps; ++w) {
        const uint32_t c = counts[w * width + row];
        counts[w * width + row] = (unsigned short)total[j];
        total[j] += c;
      }
    }
  }
  const uint32_t at = before + scan_block(total[0] + total[1], warp_sums, all);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t row = threadIdx.x * 2 + j;
    if (row < mine) p.starts[slots + row] = first[row] = j == 0 ? at : at + total[0];
  }
  if (me == kSortBlocks - 1 && threadIdx.x == 0) p.starts[p.rows] = before + all;
  __syncthreads();
  auto put = [&](const uint32_t to, const uint32_t key, const uint32_t pos) {
    p.key_out[to] = key;
    p.pos_out[to] = pos;
  };
  if (warp < (int)warps) {
    if (rounds == 1) {
      if (only_rank != ~0u) put(first[only_key / kSortBlocks] + my_counts[only_key / kSortBlocks] + only_rank, only_key, only_pos);
    } else {  // the counters now say where the warp's tokens begin: counting on gives each its place
      walk(std::true_type{}, [&](const uint32_t key, const uint32_t rank, const uint32_t pos) { put(first[key / kSortBlocks] + rank, key, pos); });
    }
  }
}

// More tokens, or more rows: least digit first, three launches per digit.
struct RadixParams {
  const void* ids;
  uint32_t* key_in;        // of the first digit, written by the counting from the ids, which are read once: the passes agree whatever another stream does to them
  const uint32_t* pos_in;  // null: the tokens in their order
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* hist;   // [bin][block]
  uint32_t* total;  // [bin]
  uint32_t n, rows, blocks;
  int32_t ids_bits, shift, digit_bits;
};
__global__ void __launch_bounds__(kRadixThreads) radix_count_kernel(const __grid_constant__ RadixParams p) {
  chain_wait();
  chain_release();
  __shared__ uint32_t count[kBinsMax];
  for (int i = threadIdx.x; i < kBinsMax; i += kRadixThreads) count[i] = 0;
  __syncthreads();
  const uint32_t mask = (1u << p.digit_bits) - 1u;
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) {
    const unsigned long long i = (unsigned long long)blockIdx.x * kRadixTile + r * kRadixThreads + threadIdx.x;
    if (i < p.n) {
      const uint32_t key = p.shift == 0 ? key_of(id_at(p.ids, p.ids_bits, i), p.rows) : p.key_in[i];
      if (p.shift == 0) p.key_in[i] = key;
      atomicAdd(&count[(key >> p.shift) & mask], 1u);
    }
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
  __shared__ uint32_t warp_sums[kRadixThreads / 32];
  static_assert(kRadixThreads == kBinsMax, "a thread per digit");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t i = threadIdx.x; i < sizeof(counts) / 4; i += kRadixThreads) ((uint32_t*)counts)[i] = 0;
  __syncthreads();
  const uint32_t mask = (1u << p.digit_bits) - 1u;
  const unsigned long long i0 = (unsigned long long)blockIdx.x * kRadixTile + warp * (kRadixRounds * 32) + lane;
  uint32_t key[kRadixRounds], rank[kRadixRounds];
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) key[r] = i0 + r * 32 < p.n ? p.key_in[i0 + r * 32] : 0u;
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) rank[r] = rank_in_warp((key[r] >> p.shift) & mask, i0 + r * 32 < p.n, p.digit_bits, counts[warp], lane);
  __syncthreads();
  uint32_t sum = 0;
#pragma unroll 4
  for (int w = 0; w < kRadixThreads / 32; ++w) {
    const uint32_t c = counts[w][threadIdx.x];
    counts[w][threadIdx.x] = (unsigned short)sum;
    sum += c;
  }
  uint32_t all;
  const uint32_t smaller = scan_block(threadIdx.x <= mask ? p.total[threadIdx.x] : 0u, warp_sums, all);
  base[threadIdx.x] = smaller + p.hist[(unsigned long long)threadIdx.x * p.blocks + blockIdx.x];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRadixRounds; ++r) {
    if (i0 + r * 32 < p.n) {
      const uint32_t digit = (key[r] >> p.shift) & mask, to = base[digit] + counts[warp][digit] + rank[r];
      p.key_out[to] = key[r];
      p.pos_out[to] = p.pos_in != nullptr ? p.pos_in[i0 + r * 32] : (uint32_t)(i0 + r * 32);
    }
  }
}

// Where the tokens of each row begin in the sorted order: a search per row.
constexpr int kStartsThreads = 256;
__global__ void __launch_bounds__(kStartsThreads) starts_kernel(const uint32_t* key, const uint32_t n, const uint32_t rows, uint32_t* starts, uint32_t* counters, const uint32_t n_counters) {
  chain_wait();
  chain_release();
  const uint32_t i = blockIdx.x * kStartsThreads + threadIdx.x;
  for (uint32_t c = i; c < n_counters; c += gridDim.x * kStartsThreads) counters[c] = 0;
  if (i > rows) return;
  uint32_t lo = 0, hi = n;  // the first token whose key is at least i
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (key[mid] < i) lo = mid + 1; else hi = mid;
  }
  starts[i] = lo;
}

// ---- (2) the sums ----------------------------------------------------------------------------------------------------
struct SumParams {
  const void* dy;
  const uint32_t* key;
  const uint32_t* pos;
  const uint32_t* starts;
  uint32_t* counters;  // [3][chunk][tile]
  void* out;
  float* partial;  // [chunk][first, last row][tiles * kTileCols]
  unsigned long long dim;
  unsigned long long row_bytes;  // of the gradient
  uint32_t dy_bytes;             // between rows of dY
  uint32_t rows, last_token, tiles, chunk, chunks;
  uint32_t lead, sum_blocks, block_rows;  // rows that a warp of the sums clears, blocks of the sums, and rows that a block behind them clears
  int32_t dealt;  // starts is in the order of slot_of, not of the rows
  float factor;
  Drop drop;
};

// Which of up to 32 rows from r on have no token.
FO_DEVI uint32_t rows_without_tokens(const SumParams& p, const uint32_t r, const uint32_t end, const int lane) {
  const uint32_t mine = min(r + lane, end - 1), s = p.dealt ? slot_of(mine, p.rows) : mine;
  return __ballot_sync(~0u, r + lane < end && p.starts[s] == p.starts[s + 1]);
}

constexpr int kClearThreads = kSumThreads;
static_assert(kClearThreads == 8 * 32, "eight warps share 32 rows");
// Rows that a block clears: long ones, one or more a warp, of about 1 / 8 of what an SM has to clear, 4 KB to `most` bytes; or a group of 32 short ones a warp.  The fewer blocks an SM
// holds, the more a block has to do: 128256 rows of 8 KB and 66 tokens 149 us with 64 KB a block (three blocks of sum_kernel an SM), 150 with 128, 153 with 256; with dropout (two)
// 161, 150, 152; 200000 rows of 2000 bytes 82 and 98 with 32 KB, 70 and 77 with 64, 70 and 74 with 128.
constexpr int clear_bytes_most(const bool drop) { return drop ? 131072 : 65536; }
static uint32_t rows_to_clear(const unsigned long long rows, const unsigned long long row_bytes, const unsigned long long most) {
  unsigned long long bytes = rows * row_bytes / (8 * kSms);
  bytes = bytes < 4096 ? 4096 : (bytes < most ? bytes : most);
  return row_bytes >= kLongRow ? (uint32_t)((bytes / row_bytes + 7) / 8 * 8 + (bytes < row_bytes ? 8 : 0)) : kClearThreads;
}

// Rows that a warp of the sums with dropout clears, a few behind every four tokens, before blocks of their own clear what is left: its time goes into draws, which leave the memory idle, and
// two such blocks leave no room on an SM for a third that clears.  16384 tokens of 768 bf16 columns into 50257 rows 34.4 us with 24 KB a warp, 38.8 with none, 35.9 with 16, 35.4 with 32 (the
// blocks behind fill the time until the last sums are done); 60000 67.0, 70.9, 66.6, 70.2.  Without dropout three blocks share an SM and the sums wait for the memory: nothing gained.
constexpr unsigned long long kLeadBytes = 24576;
static uint32_t lead_rows(const unsigned long long rows, const unsigned long long row_bytes, const unsigned long long warps, const bool drop) {
  if (!drop || row_bytes < kLongRow) return 0;
  const unsigned long long share = (rows + warps - 1) / warps, most = kLeadBytes / row_bytes, lead = share < most ? share : most;
  return (uint32_t)(lead < 32 ? lead : 32);
}

// Clears the rows without a token from r0 to r1 - 1, by a block: 32 rows at a time that the warps share where they are long, else each warp has its own.
FO_DEVI void clear_block(const SumParams& p, const uint32_t r0, const uint32_t r1, const int lane, const int warp) {
  const bool shared = p.row_bytes >= kLongRow;
  for (uint32_t r = shared ? r0 : r0 + warp * 32; r < r1; r += shared ? 32 : kClearThreads) {
    uint32_t empty = rows_without_tokens(p, r, r1, lane);
    if (shared) empty &= 0x01010101u << warp;
    clear_rows((char*)p.out + r * p.row_bytes, min(32u, r1 - r), empty, p.row_bytes, lane);
  }
}

// A lane's eight columns of a row of the gradient, `to` being where they begin: neighbours, or every 32nd, so that neighbours lie in neighbouring
// lanes (`count`: columns from the lane's first one to the end of the tile).
template <int OT, bool VECTORS>
FO_DEVI void write_row(char* to, const int count, const float (&v)[8]) {
  if constexpr (VECTORS) {
    Oct<OT> o;
    o.set(v);
    if (count > 0) o.store(to);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 < count) store1<OT>(to, j * 32, v[j]);
  }
}

FO_DEVI void put8(float* to, const float (&v)[8]) {
  __stcg((float4*)to, make_float4(v[0], v[1], v[2], v[3]));
  __stcg((float4*)to + 1, make_float4(v[4], v[5], v[6], v[7]));
}
// Where the partial sum of a chunk's first row (begun in an earlier chunk) or last row (going on in the next) lies.
FO_DEVI float* piece_at(const SumParams& p, const uint32_t chunk, const bool last, const uint32_t tile, const int lane) {
  return p.partial + (((unsigned long long)chunk * 2 + (last ? 1 : 0)) * p.tiles + tile) * kTileCols + lane * 8;
}
// The pieces of a row whose tokens lie in the chunks c0 ... c1, as `chunk`, one of them, sees them.  They are added up in groups of about the square root of their
// number by the last of each to come, the groups by the last of those, in the order of the tokens whoever comes last: the sum does not depend on
// it.  (One warp adding up 500 pieces would take longer than everything else.)
struct Pieces {
  uint32_t c0, pieces, group, groups, from, end;  // from ... end - 1: the chunk's group
  uint32_t* counter;                              // of the group
};
FO_DEVI Pieces pieces_of(const SumParams& p, const uint32_t chunk, const uint32_t c0, const uint32_t c1, const uint32_t tile) {
  Pieces r;
  r.c0 = c0;
  r.pieces = c1 - c0 + 1;
  r.group = max(16u, (uint32_t)ceilf(sqrtf((float)r.pieces)));
  const uint32_t g = (chunk - c0) / r.group;
  r.groups = (r.pieces + r.group - 1) / r.group;
  r.from = g * r.group;
  r.end = min(r.from + r.group, r.pieces);
  // (a chunk may hold the first piece of one row and begin a group of another: they count apart)
  r.counter = p.counters + (g == 0 ? 0u : p.chunks * p.tiles) + (c0 + r.from) * p.tiles + tile;
  return r;
}
// The whole sum of a row in `sum` (true), once all pieces of the chunk's group are there, if that was the last group.
FO_DEVI bool join_pieces(const SumParams& p, const Pieces& r, const uint32_t tile, const int lane, float (&sum)[8]) {
  uint32_t from = r.from, end = r.end, step = 1;
#pragma unroll 1
  for (int level = 0;; ++level) {
    __threadfence();
    float4 t[2] = {};
#pragma unroll 1
    for (uint32_t i = from; i < end; i += 4 * step) {
      float4 a[4][2];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * step < end) {
          const float4* const at = (const float4*)piece_at(p, r.c0 + i + u * step, i + u * step == 0, tile, lane);
          a[u][0] = __ldcg(at);
          a[u][1] = __ldcg(at + 1);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * step < end) {
#pragma unroll
          for (int h = 0; h < 2; ++h) t[h] = make_float4(fadd(t[h].x, a[u][h].x), fadd(t[h].y, a[u][h].y), fadd(t[h].z, a[u][h].z), fadd(t[h].w, a[u][h].w));
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[4 * h] = t[h].x; sum[4 * h + 1] = t[h].y; sum[4 * h + 2] = t[h].z; sum[4 * h + 3] = t[h].w;
    }
    if (level == 1 || r.groups == 1) return true;
    put8(piece_at(p, r.c0 + from, from == 0, tile, lane), sum);
    __threadfence();
    __syncwarp();
    uint32_t seen = 0;
    if (lane == 0) seen = atomicAdd(p.counters + 2 * p.chunks * p.tiles + r.c0 * p.tiles + tile, 1u);
    if (__shfl_sync(~0u, seen, 0) + 1 != r.groups) return false;
    from = 0; end = r.pieces; step = r.group;
  }
}

// A tile of a row of DT elements in shared memory.  VECTORS: eight neighbouring elements per lane, which copies and reads its own; otherwise every 32nd, and
// the tile comes as the 16 bytes each that hold it, as far into them as it is in memory.
struct Bounds {  // of the array: nothing outside is touched
  const char *lo, *hi;
};
template <int DT, bool VECTORS>
struct Tile {
  static constexpr int kBytes = kTileCols * size_of(DT) + (VECTORS ? 0 : 16);
  // `from`: where the tile's first column lies
  static FO_DEVI void fetch(unsigned char* stage, const char* from, const int columns, const int lane, const Bounds in) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(stage);
    if constexpr (VECTORS) {
      if (lane * 8 < columns) {
        copy_async16(to + lane * 16, from + lane * 8 * size_of(DT));
        if constexpr (DT == FO_F32) copy_async16(to + 512 + lane * 16, from + lane * 32 + 16);
      }
    } else {
      const int into = (int)((uintptr_t)from & 15), size = (into + columns * size_of(DT) + 15) & ~15;
      const char* const a = from - into;
      if (a < in.lo || a + size > in.hi) {
        for (int e = lane; e < columns; e += 32) {
          if constexpr (DT == FO_F32) ((uint32_t*)(stage + into))[e] = ((const uint32_t*)from)[e];
          else ((unsigned short*)(stage + into))[e] = ((const unsigned short*)from)[e];
        }
      } else {
#pragma unroll
        for (int c = 0; c < (kBytes + 511) / 512; ++c)
          if (c * 512 + lane * 16 < size) copy_async16(to + c * 512 + lane * 16, a + c * 512 + lane * 16);
      }
    }
  }
  static FO_DEVI void get(const unsigned char* stage, const char* from, const int lane, float (&v)[8]) {
    if constexpr (VECTORS) {
      Oct<DT> x;
      x.a = *(const uint4*)(stage + lane * 16);
      if constexpr (DT == FO_F32) x.b = *(const uint4*)(stage + 512 + lane * 16);
      x.get(v);
    } else {
      const unsigned char* const at = stage + ((uintptr_t)from & 15);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = load1<DT>(at, j * 32 + lane);
    }
  }
};

// Bound by HBM: every row of dY is read once, in pieces of 512 bytes (1 KB in fp32) wherever the sort has put it.  A warp copies the pieces of the
// next tokens into a ring in shared memory while it adds those at hand; where the gradient is added to, also what lies in the rows that begin among
// them, which the sums start from.
template <int DT, int OT, bool VECTORS, bool ACC>
struct Ring {
  static constexpr int kStages = DT == FO_F32 || ACC ? 4 : 8;
  static constexpr int kOld = Tile<DT, VECTORS>::kBytes, kStage = kOld + (ACC ? Tile<OT, VECTORS>::kBytes : 0);
  static constexpr int kWarp = kStages * kStage, kBlock = kWarp * (kSumThreads / 32);
};
template <int DT, int OT, bool VECTORS, bool DROP, bool ACC>
__global__ void __launch_bounds__(kSumThreads, sum_blocks_per_sm(DROP)) sum_kernel(const __grid_constant__ SumParams p) {
  chain_wait();
  chain_release();
  using R = Ring<DT, OT, VECTORS, ACC>;
  constexpr int kStages = R::kStages;
  extern __shared__ __align__(16) unsigned char rings[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const unsigned long long task = (unsigned long long)blockIdx.x * (kSumThreads / 32) + warp;
  if constexpr (!ACC) {
    if (blockIdx.x >= p.sum_blocks) {
      const unsigned long long r0 = (unsigned long long)p.sum_blocks * (kSumThreads / 32) * p.lead + (unsigned long long)(blockIdx.x - p.sum_blocks) * p.block_rows;
      if (r0 < p.rows) clear_block(p, (uint32_t)r0, (uint32_t)min(r0 + p.block_rows, (unsigned long long)p.rows), lane, warp);
      return;
    }
  }
  const uint32_t tile = (uint32_t)(task % p.tiles), chunk = (uint32_t)(task / p.tiles);
  // The warp's share of the first rows, a lane's where its tokens begin and end: asked for here, looked at when the first tokens are on their way.
  uint32_t lead_begins = 0, lead_ends = 1, to_clear = 0;
  char* lead = nullptr;
  if constexpr (DROP && !ACC) {
    const unsigned long long r0 = task * p.lead, r = r0 + lane;
    if ((uint32_t)lane < p.lead && r < p.rows) {
      const uint32_t s = p.dealt ? slot_of((uint32_t)r, p.rows) : (uint32_t)r;
      lead_begins = p.starts[s];
      lead_ends = p.starts[s + 1];
    }
    lead = (char*)p.out + r0 * p.row_bytes;
  }
  const auto clear_lead = [&](uint32_t most) {
    if constexpr (DROP && !ACC) {
      for (; to_clear != 0 && most != 0; to_clear &= to_clear - 1u, --most) {
        char* const at = lead + (unsigned long long)(__ffs(to_clear) - 1) * p.row_bytes;
        clear_bytes(at, at + p.row_bytes, lane);
      }
    }
  };
  const auto clear_all = [&]() {
    if constexpr (DROP && !ACC) to_clear = __ballot_sync(~0u, lead_begins == lead_ends);
    clear_lead(32);
  };
  if (chunk >= p.chunks) {
    clear_all();
    return;
  }
  const uint32_t first = (uint32_t)((unsigned long long)chunk * p.chunk);
  // keys and places of 32 tokens, one per lane; what lies behind the last token that names a row is nothing
  const uint32_t n = p.starts[p.rows];
  uint32_t key = first + lane <= p.last_token ? p.key[first + lane] : 0u, pos = first + lane <= p.last_token ? p.pos[first + lane] : 0u;
  if (first >= n) {
    clear_all();
    return;
  }
  const uint32_t end = (uint32_t)min((unsigned long long)first + p.chunk, (unsigned long long)n);
  const uint32_t last_row = p.key[end - 1];
  const unsigned long long c0 = (unsigned long long)tile * kTileCols;
  const int columns = p.dim - c0 < kTileCols ? (int)(p.dim - c0) : kTileCols;  // of this tile
  const int count = columns - (VECTORS ? lane * 8 : lane);
  const char* const from = (const char*)p.dy + c0 * size_of(DT);
  char* const out = (char*)p.out + c0 * size_of(OT);
  constexpr int kLaneOut = (VECTORS ? 8 : 1) * size_of(OT);
  unsigned char* const ring = rings + warp * R::kWarp;
  uint32_t row = __shfl_sync(~0u, key, 0);
  const uint32_t first_row = row;
  const uint32_t slot = p.dealt ? slot_of(row, p.rows) : row, row_begins = p.starts[slot], row_ends = p.starts[slot + 1];
  const uint32_t last_ends = p.starts[(p.dealt ? slot_of(last_row, p.rows) : last_row) + 1];
  const uint2 off = DROP ? drop_offset(p.drop) : make_uint2(0u, 0u);
  bool opened = row_begins < first;  // in an earlier chunk
  auto heads_of = [&](const uint32_t keys, const uint32_t before) {  // bit k: a row begins with token k of the 32
    const uint32_t left = __shfl_up_sync(~0u, keys, 1);
    return __ballot_sync(~0u, keys != (lane == 0 ? before : left));
  };
  uint32_t heads = heads_of(key, opened ? row : ~0u), next_key = 0, next_pos = 0, next_heads = 0;
  const Bounds dy_in = {(const char*)p.dy, (const char*)p.dy + (unsigned long long)p.last_token * p.dy_bytes + p.dim * size_of(DT)};
  const Bounds out_in = {(const char*)p.out, (const char*)p.out + p.rows * p.row_bytes};
  // token `t` of the 64 at hand into a stage
  auto fetch = [&](const uint32_t t, const uint32_t at, const int stage) {
    unsigned char* const to = ring + stage * R::kStage;
    Tile<DT, VECTORS>::fetch(to, from + (unsigned long long)at * p.dy_bytes, columns, lane, dy_in);
    if constexpr (ACC) {
      const uint32_t r = __shfl_sync(~0u, t < 32 ? key : next_key, t & 31);
      if (((t < 32 ? heads : next_heads) >> (t & 31) & 1u) != 0)
        Tile<OT, VECTORS>::fetch(to + R::kOld, out + r * p.row_bytes, columns, lane, out_in);
    }
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) {
    const uint32_t at = __shfl_sync(~0u, pos, k);
    if (first + k < end) fetch(k, at, k);
    copy_commit();
  }
  if constexpr (DROP && !ACC) to_clear = __ballot_sync(~0u, lead_begins == lead_ends);
  const uint32_t groups = (end - first + 3) / 4, at_once = (__popc(to_clear) + groups - 1) / groups;
  float sum[8] = {};
  bool any = false;  // a row began in this chunk
  // Four tokens at a time: single ones cost a third more instructions, and with the draws of dropout in it, the loop unrolled over eight outgrew
  // the instruction cache.
  static_assert(kStages % 4 == 0 && kStages <= 8, "a group of four lies in stages 0-3 or 4-7");
#pragma unroll 1
  for (uint32_t here = first; here < end; here += 32) {
    next_key = here + 32 + lane < end ? p.key[here + 32 + lane] : 0u;
    next_pos = here + 32 + lane < end ? p.pos[here + 32 + lane] : 0u;
#pragma unroll 1
    for (uint32_t k0 = 0; k0 < 32; k0 += 4) {
      if (here + k0 >= end) break;
      if (k0 == (kStages == 8 ? 24 : 28)) next_heads = heads_of(next_key, __shfl_sync(~0u, key, 31));
      const uint32_t half = kStages == 8 ? k0 & 4u : 0u;
      unsigned char* const group = ring + half * R::kStage;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t k = k0 + s, a = k + kStages - 1;
        if (here + k >= end) break;
        copy_wait<kStages - 2>();
        if constexpr (!VECTORS) __syncwarp();  // the other lanes' copies are there, and the stage that is filled next has been read
        const uint32_t ahead = __shfl_sync(~0u, a < 32 ? pos : next_pos, a & 31);
        // the stage that is filled next: the one behind, of this group or the last of the other
        if (here + a < end) fetch(a, ahead, kStages == 8 ? (s == 0 ? (int)(half ^ 4u) + 3 : (int)half + s - 1) : (s + 3) % 4);
        copy_commit();
        const uint32_t at = DROP || !VECTORS ? __shfl_sync(~0u, pos, k) : 0u;
        const unsigned long long e0 = at * p.dim + c0;
        uint4 w = {};
        if constexpr (DROP && VECTORS) w = draw8(p.drop, off, (unsigned long long)at * (uint32_t)(p.dim / 8) + (tile * (kTileCols / 8) + lane));
        const unsigned char* const stage = group + s * R::kStage;
        if ((heads >> k & 1u) != 0) {  // (the same for the whole warp)
          if (opened) put8(piece_at(p, chunk, false, tile, lane), sum);
          else if (any) write_row<OT, VECTORS>(out + row * p.row_bytes + lane * kLaneOut, count, sum);
          any = true;
          opened = false;
          row = __shfl_sync(~0u, key, k);
          if constexpr (ACC) {
            Tile<OT, VECTORS>::get(stage + R::kOld, out + row * p.row_bytes, lane, sum);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
          }
        }
        float v[8];
        Tile<DT, VECTORS>::get(stage, from + (unsigned long long)at * p.dy_bytes, lane, v);
        if constexpr (DROP && VECTORS) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (stays(p.drop, w, j)) sum[j] = __fmaf_rn(v[j], p.factor, sum[j]);
        } else if constexpr (DROP) {  // the warp's 256 columns lie in 32 or 33 blocks of eight
          const uint32_t skew = (uint32_t)e0 & 7u;
          const uint32_t low = keep8(p.drop, off, (e0 >> 3) + lane), high = skew != 0 ? keep8(p.drop, off, (e0 >> 3) + 32) : 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t e = skew + j * 32 + lane;
            const uint32_t bits = __shfl_sync(~0u, low, (e >> 3) & 31);
            if (((e >= 256 ? high : bits) >> (e & 7) & 1u) != 0) sum[j] = __fmaf_rn(v[j], p.factor, sum[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] = __fmaf_rn(v[j], p.factor, sum[j]);
        }
      }
      clear_lead(at_once);
    }
    key = next_key;
    pos = next_pos;
    heads = next_heads;
  }
  const bool goes_on = last_ends > end;
  if (opened) put8(piece_at(p, chunk, false, tile, lane), sum);
  else if (goes_on) put8(piece_at(p, chunk, true, tile, lane), sum);
  else write_row<OT, VECTORS>(out + row * p.row_bytes + lane * kLaneOut, count, sum);
  // The pieces: of the row that began earlier (lane 0 counts), and of the one that goes on (lane 1).
  const bool first_left = row_begins < first, last_left = !opened && goes_on;
  if (!first_left && !last_left) return;
  __threadfence();
  __syncwarp();
  bool came_last = false;
  if (lane == 0 ? first_left : lane == 1 && last_left) {
    const Pieces r = pieces_of(p, chunk, lane == 0 ? row_begins / p.chunk : chunk, ((lane == 0 ? row_ends : last_ends) - 1) / p.chunk, tile);
    came_last = atomicAdd(r.counter, 1u) + 1 == r.end - r.from;
  }
  const uint32_t to_join = __ballot_sync(~0u, came_last);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if ((to_join >> which & 1u) == 0) continue;
    const Pieces r = pieces_of(p, chunk, which == 0 ? row_begins / p.chunk : chunk, ((which == 0 ? row_ends : last_ends) - 1) / p.chunk, tile);
    if (join_pieces(p, r, tile, lane, sum)) write_row<OT, VECTORS>(out + (which == 0 ? first_row : last_row) * p.row_bytes + lane * kLaneOut, count, sum);
  }
}

// ---- a handful of tokens, in one launch -------------------------------------------------------------------------------
// Every block reads all ids.  A warp per token and 256 columns sees whether its token is the first with its id, and then adds up the rows of all that
// have it, in their order; the blocks behind clear the rows that none names.  Bound by launching and by the latency of ids and rows, which the three
// launches above pay several times (64 tokens of 1024 fp32 columns into 8192 rows, 33.6 MB: 7.6 us; 65 through them 12.3).  A row of k tokens takes k / 4 trips
// to memory, so it ends at 64.
struct FewParams {
  const void* dy;
  const void* ids;
  char* out;
  unsigned long long dim, row_bytes, dy_bytes;
  uint32_t n, rows, tiles, token_blocks, clear_rows;
  int32_t ids_bits, out_dtype, accumulate;
  float factor;
  Drop drop;
};
template <int DT, bool VECTORS>
__global__ void __launch_bounds__(kSumThreads) few_kernel(const __grid_constant__ FewParams p) {
  chain_wait();
  chain_release();
  extern __shared__ uint32_t named[];  // a bit per row of the block
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  uint32_t key[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) key[h] = h * 32 + lane < p.n ? key_of(id_at(p.ids, p.ids_bits, h * 32 + lane), p.rows) : p.rows;
  if (blockIdx.x >= p.token_blocks) {
    const uint32_t r0 = (blockIdx.x - p.token_blocks) * p.clear_rows, r1 = min(r0 + p.clear_rows, p.rows);
    for (uint32_t i = threadIdx.x; i < (r1 - r0 + 31) / 32; i += kSumThreads) named[i] = 0;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (key[h] >= r0 && key[h] < r1) atomicOr(&named[(key[h] - r0) / 32], 1u << ((key[h] - r0) & 31));
    }
    __syncthreads();
    const bool shared = p.row_bytes >= kLongRow;  // (as in clear_block)
    for (uint32_t r = shared ? r0 : r0 + warp * 32; r < r1; r += shared ? 32 : kSumThreads) {
      uint32_t empty = ~named[(r - r0) / 32];
      if (shared) empty &= 0x01010101u << warp;
      if (r1 - r < 32) empty &= (1u << (r1 - r)) - 1u;
      clear_rows(p.out + r * p.row_bytes, min(32u, r1 - r), empty, p.row_bytes, lane);
    }
    return;
  }
  const uint32_t task = blockIdx.x * (kSumThreads / 32) + warp, token = task / p.tiles, tile = task - token * p.tiles;
  if (token >= p.n) return;
  const uint32_t mine_low = __shfl_sync(~0u, key[0], token & 31), mine_high = __shfl_sync(~0u, key[1], token & 31), row = token < 32 ? mine_low : mine_high;
  if (row >= p.rows) return;
  const uint32_t same_low = __ballot_sync(~0u, key[0] == row), same_high = __ballot_sync(~0u, key[1] == row);
  unsigned long long same = (unsigned long long)same_high << 32 | same_low;
  if ((same & ((1ull << token) - 1ull)) != 0) return;  // another has it
  const uint2 off = drop_offset(p.drop);
  const unsigned long long c0 = (unsigned long long)tile * kTileCols;
  const int columns = p.dim - c0 < kTileCols ? (int)(p.dim - c0) : kTileCols, count = columns - (VECTORS ? lane * 8 : lane);
  const char* const from = (const char*)p.dy + (c0 + (VECTORS ? lane * 8 : lane)) * size_of(DT);
  constexpr int kAhead = 4;
  float sum[8] = {};
  while (same != 0) {
    float v[kAhead][8];
    uint32_t at[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      at[k] = same != 0 ? (uint32_t)__ffsll((long long)same) - 1u : ~0u;
      same &= same - 1ull;
      const char* const x = from + at[k] * p.dy_bytes;
      if (at[k] == ~0u) continue;
      if constexpr (VECTORS) {
        Oct<DT> o;
        if (count > 0) {
          o.load(x);
          o.get(v[k]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j * 32 < count) v[k][j] = load1<DT>(x, j * 32);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (at[k] == ~0u) break;
      const unsigned long long e0 = at[k] * p.dim + c0;
      uint32_t low = 0xFFu, high = 0xFFu;
      if (p.drop.on) {
        low = keep8(p.drop, off, (e0 >> 3) + lane);
        if ((e0 & 7) != 0) high = keep8(p.drop, off, (e0 >> 3) + 32);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t keep = low >> j;
        if constexpr (!VECTORS) {
          const uint32_t e = ((uint32_t)e0 & 7u) + j * 32 + lane, bits = __shfl_sync(~0u, low, (e >> 3) & 31);
          keep = (e >= 256 ? high : bits) >> (e & 7);
        }
        if (!p.drop.on || (keep & 1u) != 0) sum[j] = __fmaf_rn(v[k][j], p.factor, sum[j]);
      }
    }
  }
  auto write = [&](auto tag) {
    constexpr int OT = decltype(tag)::value;
    char* const to = p.out + row * p.row_bytes + (c0 + (VECTORS ? lane * 8 : lane)) * size_of(OT);
    if (p.accumulate) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        constexpr int kStep = VECTORS ? 1 : 32;
        if (VECTORS ? count > 0 : j * 32 < count) sum[j] = fadd(load1<OT>(to, j * kStep), sum[j]);
      }
    }
    write_row<OT, VECTORS>(to, count, sum);
  };
  if (p.out_dtype == FO_F32) write(std::integral_constant<int, FO_F32>{});
  else if (p.out_dtype == FO_BF16) write(std::integral_constant<int, FO_BF16>{});
  else write(std::integral_constant<int, FO_F16>{});
}

static int few_tokens(const FoEmbedGrad& f, const SumParams& s, const bool vectors, cudaStream_t stream) {
  FewParams p = {};
  p.dy = f.dy; p.ids = f.ids; p.out = (char*)f.out;
  p.dim = f.dim; p.row_bytes = s.row_bytes; p.dy_bytes = s.dy_bytes;
  p.n = (uint32_t)f.n_tokens; p.rows = s.rows; p.tiles = s.tiles;
  p.ids_bits = f.ids_bits; p.out_dtype = f.out_dtype; p.accumulate = f.accumulate != 0;
  p.factor = s.factor; p.drop = s.drop;
  p.token_blocks = (p.n * p.tiles + kSumThreads / 32 - 1) / (kSumThreads / 32);
  unsigned int grid = p.token_blocks;
  if (!f.accumulate) {
    p.clear_rows = rows_to_clear(s.rows, s.row_bytes, 32768);
    grid += (p.rows + p.clear_rows - 1) / p.clear_rows;
  }
  if (grid == 0) return FO_OK;
  void (*kernel)(const FewParams) = nullptr;
#define X(D) \
  if (f.dy_dtype == D) kernel = vectors ? few_kernel<D, true> : few_kernel<D, false>;
  X(FO_F32) X(FO_BF16) X(FO_F16)
#undef X
  bool chained = true;
  const cudaError_t e = launch_chained(kernel, grid, (unsigned int)kSumThreads, (int)((p.clear_rows + 31) / 32 * 4), chained, stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
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

static int sort_by_rows(const FoEmbedGrad& f, const GradPlan& g, cudaStream_t stream) {
  char* const ws = (char*)f.workspace;
  const uint32_t n = (uint32_t)f.n_tokens, rows = (uint32_t)f.rows, n_counters = 3 * g.chunks * g.tiles;
  uint32_t *const key = (uint32_t*)(ws + g.key[0]), *const pos = (uint32_t*)(ws + g.pos[0]), *const starts = (uint32_t*)(ws + g.starts), *const counters = (uint32_t*)(ws + g.counters);
  int row_bits = 0;
  while (rows / kSortBlocks >> row_bits != 0) ++row_bits;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(FO_ERR_CUDA, "fo_embed_grad: cannot query the current device");
  if (dev >= 64 || (ready.load() >> dev & 1) == 0) {
    if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) != cudaSuccess ||
        cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem) != cudaSuccess)
      return fail(FO_ERR_CUDA, "fo_embed_grad: cannot set the shared memory size");
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  bool chained = true;
  cudaError_t e;
  if (g.alone) {
    const SortParams p = {f.ids, key, pos, starts, counters, n, rows, n_counters, f.ids_bits, row_bits};
    e = launch_chained(sort_kernel, kSortBlocks, (unsigned int)kSortThreads, (int)g.sort_smem, chained, stream, p);
  } else {
    const DealParams p = {f.ids, (uint32_t*)(ws + g.key[1]), (uint32_t*)(ws + g.pos[1]), (uint32_t*)(ws + g.hist), key, pos, starts, counters, n, rows,
                          (n + kDealTokens - 1) / kDealTokens, n_counters, f.ids_bits, row_bits};
    e = launch_chained(deal_kernel, p.blocks, (unsigned int)kSortThreads, 0, chained, stream, p);
    if (e == cudaSuccess) e = launch_chained(order_kernel, kSortBlocks, (unsigned int)kSortThreads, (int)g.sort_smem, chained, stream, p);
  }
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}

// The sort over several launches; key[result] and pos[result] hold what comes of it.
static int sort_in_memory(const FoEmbedGrad& f, const GradPlan& g, cudaStream_t stream, int& result) {
  char* const ws = (char*)f.workspace;
  RadixParams p = {};
  int passes;
  digits((uint32_t)f.rows, passes, p.digit_bits);
  p.ids = f.ids; p.ids_bits = f.ids_bits;
  p.hist = (uint32_t*)(ws + g.hist); p.total = (uint32_t*)(ws + g.total);
  p.n = (uint32_t)f.n_tokens; p.rows = (uint32_t)f.rows; p.blocks = g.blocks;
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < passes && e == cudaSuccess; ++pass) {
    p.key_in = (uint32_t*)(ws + g.key[(pass + 1) & 1]);
    p.pos_in = pass == 0 ? nullptr : (const uint32_t*)(ws + g.pos[(pass - 1) & 1]);
    p.key_out = (uint32_t*)(ws + g.key[pass & 1]); p.pos_out = (uint32_t*)(ws + g.pos[pass & 1]);
    p.shift = pass * p.digit_bits;
    result = pass & 1;
    bool chained = true;
    e = launch_chained(radix_count_kernel, p.blocks, (unsigned int)kRadixThreads, 0, chained, stream, p);
    if (e == cudaSuccess) e = launch_chained(radix_scan_kernel, 1u << p.digit_bits, (unsigned int)kRadixScanThreads, 0, chained, stream, p);
    if (e == cudaSuccess) e = launch_chained(radix_scatter_kernel, p.blocks, (unsigned int)kRadixThreads, 0, chained, stream, p);
  }
  bool chained = true;
  if (e == cudaSuccess)
    e = launch_chained(starts_kernel, (unsigned int)(f.rows / kStartsThreads + 1), (unsigned int)kStartsThreads, 0, chained, stream, (const uint32_t*)(ws + g.key[result]), p.n, p.rows,
                       (uint32_t*)(ws + g.starts), (uint32_t*)(ws + g.counters), (uint32_t)(3 * g.chunks * g.tiles));
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}

}  // namespace fo

using namespace fo;

extern "C" int fo_embed_grad_workspace(uint64_t rows, uint64_t dim, uint64_t n_tokens, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad_workspace: null pointer");
  *bytes = 0;
  if (int rc = sizes_ok("fo_embed_grad_workspace", rows, dim, n_tokens)) return rc;
  if (rows != 0 && dim != 0) *bytes = plan_of(rows, dim, n_tokens, false).bytes;
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
  if (!make_factor(f->scale, factor, p.factor)) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: scale %g with p = %g (scale / (1 - p) has to be 0 or a normal fp32 number)", f->scale, f->dropout.p);
  if (int rc = sizes_ok("fo_embed_grad", f->rows, f->dim, f->n_tokens)) return rc;
  if (f->rows == 0 || f->dim == 0 || (f->accumulate && f->n_tokens == 0)) return FO_OK;
  if (f->out == nullptr || (f->n_tokens > 0 && (f->ids == nullptr || f->dy == nullptr))) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: null pointer");
  if (f->dy_stride < f->dim || f->dy_stride >> 28) return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: rows %llu elements apart are %llu long", (unsigned long long)f->dy_stride, (unsigned long long)f->dim);
  const GradPlan g = plan_of(f->rows, f->dim, f->n_tokens, p.drop.on != 0);
  const unsigned long long need = plan_of(f->rows, f->dim, f->n_tokens, false).bytes;
  if (f->workspace_bytes < need || (need > 0 && (f->workspace == nullptr || !on_16_bytes(f->workspace))))
    return fail(FO_ERR_INVALID_ARG, "fo_embed_grad: a workspace of %llu bytes, aligned to 16, is needed, got %llu", need, (unsigned long long)f->workspace_bytes);
  cudaStream_t stream = (cudaStream_t)cuda_stream;
  int at = 0;
  char* const ws = (char*)f->workspace;
  p.dy = f->dy; p.out = f->out;
  p.starts = (const uint32_t*)(ws + g.starts); p.counters = (uint32_t*)(ws + g.counters);
  p.partial = (float*)(ws + g.partial);
  p.dim = f->dim; p.dy_bytes = (uint32_t)(f->dy_stride * size_of(f->dy_dtype)); p.row_bytes = f->dim * size_of(f->out_dtype);
  p.rows = (uint32_t)f->rows; p.last_token = (uint32_t)(f->n_tokens - 1); p.dealt = !g.several; p.tiles = g.tiles; p.chunk = g.chunk; p.chunks = g.chunks;
  const bool vectors = f->dim % 8 == 0 && on_16_bytes(f->dy) && f->dy_stride * size_of(f->dy_dtype) % 16 == 0 && on_16_bytes(f->out);
  if (f->n_tokens <= kFewTokens) return few_tokens(*f, p, vectors, stream);
  if (int rc = g.several ? sort_in_memory(*f, g, stream, at) : sort_by_rows(*f, g, stream)) return rc;
  p.key = (const uint32_t*)(ws + g.key[at]); p.pos = (const uint32_t*)(ws + g.pos[at]);
  void (*kernel)(const SumParams) = nullptr;
  int smem = 0;
#define Y(D, O, V, P, A) \
  if (f->dy_dtype == D && f->out_dtype == O && vectors == V && (p.drop.on != 0) == P && (f->accumulate != 0) == A) {      \
    kernel = sum_kernel<D, O, V, P, A>;                                                                                              \
    smem = Ring<D, O, V, A>::kBlock;                                                                                                 \
  }
#define X(D, O)                                                                                                          \
  Y(D, O, true, true, true) Y(D, O, true, true, false) Y(D, O, true, false, true) Y(D, O, true, false, false)             \
  Y(D, O, false, true, true) Y(D, O, false, true, false) Y(D, O, false, false, true) Y(D, O, false, false, false)
  X(FO_F32, FO_F32) X(FO_F32, FO_BF16) X(FO_F32, FO_F16) X(FO_BF16, FO_F32) X(FO_BF16, FO_BF16) X(FO_BF16, FO_F16) X(FO_F16, FO_F32) X(FO_F16, FO_BF16) X(FO_F16, FO_F16)
#undef X
#undef Y
  const unsigned long long warps_per_block = kSumThreads / 32, blocks = ((unsigned long long)g.chunks * g.tiles + warps_per_block - 1) / warps_per_block;
  p.sum_blocks = (uint32_t)blocks;
  unsigned long long grid = blocks;
  if (!f->accumulate) {
    p.lead = lead_rows(p.rows, p.row_bytes, blocks * warps_per_block, p.drop.on != 0);
    const unsigned long long led = p.lead * blocks * warps_per_block, rest = led < p.rows ? p.rows - led : 0;
    p.block_rows = rows_to_clear(rest, p.row_bytes, clear_bytes_most(p.drop.on != 0));
    grid += (rest + p.block_rows - 1) / p.block_rows;
  }
  bool chained = true;
  cudaError_t e = cudaSuccess;
  // (some rings are above the 48 KB that need no leave; it is given at each call, for whichever device is current)
  if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = launch_chained(kernel, (unsigned int)grid, (unsigned int)kSumThreads, smem, chained, stream, p);
  return e == cudaSuccess ? FO_OK : fail(FO_ERR_CUDA, "fo_embed_grad: launch failed: %s", cudaGetErrorString(e));
}
