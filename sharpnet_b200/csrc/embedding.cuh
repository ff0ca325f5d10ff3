// Embedding lookup with a scale, and its gradient summed by word in a fixed order.
//
//   forward:   y[t, :] = scale * table[i_t, :]
//   backward:  dtable[v, :] = (accumulate ? dtable[v, :] : 0) + scale * sum over {t : i_t = v} of dy[t, :]
//
// The gradient sorts the (word, token) pairs by word, stably, and adds the rows of each word in the order of their
// tokens: no floating atomics, so the same call gives the same bits.  A frequent word (Zipf: one word can hold a tenth
// of the batch) is spread over many warps: the sorted tokens are cut into chunks of equal length, a word that crosses
// a chunk's border leaves a partial sum in the scratch memory, and a second launch adds those in chunk order.
#pragma once
#include "elementwise.cuh"
#include "ptx.cuh"

namespace snb {

enum IndexType : int { INDEX_INT32 = 0, INDEX_INT64 = 1, INDEX_FP32 = 2 };

// Set in the handle's error word when a token index lies outside the table.
constexpr int kErrorTokenIndex = 2;

// The row that index `i` of a batch names, or -1 where it lies outside the table.
__device__ __forceinline__ int load_index(const void* indices, int index_type, long long i, int vocab) {
  if (index_type == INDEX_INT32) {
    const int v = static_cast<const int*>(indices)[i];
    return (v >= 0 && v < vocab) ? v : -1;
  }
  if (index_type == INDEX_INT64) {
    const long long v = static_cast<const long long*>(indices)[i];
    return (v >= 0 && v < vocab) ? static_cast<int>(v) : -1;
  }
  const float v = rintf(static_cast<const float*>(indices)[i]);       // a NaN fails every comparison
  if (!(v >= 0.0f && v < 2147483648.0f)) return -1;
  const int id = static_cast<int>(v);
  return id < vocab ? id : -1;
}

// ---------------------------------------------------------------- forward
// Block of bx x by threads: bx consecutive vectors of a row, by rows side by side, TOKENS rows per thread one after the
// other with their loads in flight together.  Bound by memory: 16384 rows of 1024 take 17.0 us (5.3 TB/s).
template <int VEC, int TOKENS>
static __global__ void __launch_bounds__(256)
embedding_fwd_kernel(const void* __restrict__ indices, int index_type, long long tokens, int vocab, int row_vecs, float scale,
                     const float* __restrict__ table, float* __restrict__ y, int* error_word) {
  pdl_prologue();
  typedef typename Pack<VEC>::type P;
  const int col = blockIdx.y * blockDim.x + threadIdx.x;
  const long long t0 = blockIdx.x * static_cast<long long>(blockDim.y * TOKENS) + threadIdx.y;
  int id[TOKENS];
  P v[TOKENS];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < TOKENS; ++k) {
    const long long t = t0 + static_cast<long long>(k) * blockDim.y;
    id[k] = t < tokens ? load_index(indices, index_type, t, vocab) : -2;
    bad |= id[k] == -1;
  }
  if (bad && col == 0) atomicOr(error_word, kErrorTokenIndex);
  if (col >= row_vecs) return;
#pragma unroll
  for (int k = 0; k < TOKENS; ++k)
    v[k] = id[k] >= 0 ? __ldg(reinterpret_cast<const P*>(table) + static_cast<long long>(id[k]) * row_vecs + col) : P();
#pragma unroll
  for (int k = 0; k < TOKENS; ++k) {
    if (id[k] == -2) continue;
    P o;
#pragma unroll
    for (int q = 0; q < VEC; ++q) lane_set(o, q, scale * lane_get(v[k], q));
    reinterpret_cast<P*>(y)[(t0 + static_cast<long long>(k) * blockDim.y) * row_vecs + col] = o;
  }
}

// n floats become zero, by the threads tid = 0 .. stride - 1.
__device__ __forceinline__ void fill_zero(long long n, float* __restrict__ p, long long tid, long long stride) {
  const long long head = min(n, static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) >> 2);
  const long long quads = (n - head) >> 2;
  for (long long i = tid; i < quads; i += stride) reinterpret_cast<float4*>(p + head)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (tid < head) p[tid] = 0.0f;
  if (head + 4 * quads + tid < n) p[head + 4 * quads + tid] = 0.0f;
}
static __global__ void __launch_bounds__(256)
fill_zero_kernel(long long n, float* __restrict__ p) {
  pdl_prologue();
  fill_zero(n, p, blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x, static_cast<long long>(gridDim.x) * blockDim.x);
}

// ---------------------------------------------------------------- rows of words that do not occur
constexpr int kSlab = 128;            // columns of one warp: 4 per lane

// Four columns of a row: one float4 (VEC = 4), or the columns lane, lane + 32, .. of the slab (VEC = 1).
template <int VEC>
__device__ __forceinline__ float4 load_cols(const float* row, int slab, int lane, int dim) {
  if (VEC == 4) {
    const int c = slab * kSlab + 4 * lane;
    return c < dim ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  float v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = slab * kSlab + lane + 32 * k;
    v[k] = c < dim ? row[c] : 0.0f;
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}
template <int VEC>
__device__ __forceinline__ void store_cols(float* row, int slab, int lane, int dim, const float4& v) {
  if (VEC == 4) {
    const int c = slab * kSlab + 4 * lane;
    if (c < dim) *reinterpret_cast<float4*>(row + c) = v;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = slab * kSlab + lane + 32 * k;
    if (c < dim) row[c] = lane_get(v, k);
  }
}

// The gradient's rows of words that do not occur are zeros (unless it is added to).  Which words occur is known after the
// first launch of the sort, so blocks that write zeros ride along with its later launches, which are bound by latency and
// leave the memory idle.  A unit: a slab of the rows of 32 words.
struct ZeroRows {
  const unsigned* present;            // a bit per word that occurs
  float* dtable;
  int vocab, dim, slabs, vec;
  long long first, last;              // the units of this launch
};
template <int VEC>
__device__ __forceinline__ void zero_words_vec(const ZeroRows& z, long long id, int lane) {
  const long long group = id / z.slabs;
  const int slab = static_cast<int>(id % z.slabs);
  const long long first = 32 * group;
  const unsigned present = __ldcg(z.present + group);
  const int words = static_cast<int>(min(32LL, z.vocab - first));
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (VEC == 4 && z.dim < kSlab) {                     // narrow rows: as many side by side as a warp's width holds
    const int quads = z.dim >> 2;
    for (int i = lane; i < words * quads; i += 32) {
      const int w = i / quads;
      if (!(present >> w & 1)) reinterpret_cast<float4*>(z.dtable + first * z.dim)[i] = zero;
    }
    return;
  }
  for (int w = 0; w < words; ++w)
    if (!(present >> w & 1)) store_cols<VEC>(z.dtable + (first + w) * z.dim, slab, lane, z.dim, zero);
}
// Warp `warp` of all warps that write zeros in this launch.
__device__ __forceinline__ void zero_words(const ZeroRows& z, long long warp, long long warps) {
  const int lane = threadIdx.x & 31;
  for (long long id = z.first + warp; id < z.last; id += warps) {
    if (z.vec) zero_words_vec<4>(z, id, lane);
    else zero_words_vec<1>(z, id, lane);
  }
}

// ---------------------------------------------------------------- stable sort of (word, token), one digit a pass
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxBits = 9;                      // digit of at most 9 bits: 16 warps x 512 counters = 32 KB
constexpr int kSortMaxBins = 1 << kSortMaxBits;
constexpr int kSortTile = 2048;                      // tokens of a block of the sort in several launches
constexpr int kSortClusterTokens = 32768;            // most tokens of the sort in one launch: eight blocks of 4096

struct SortPass {
  const void* indices;                // the caller's indices: read by the first pass in place of `in`
  int index_type, vocab, padding;
  const uint2* in;                    // (word, token)
  uint2* out;
  unsigned *counts;                   // [bins][tiles]
  unsigned *totals;                   // [bins]
  unsigned *present;                  // a bit per word that occurs, cleared before; NULL where nobody asks
  unsigned *crossing;                 // a counter of the sums, cleared here
  int n, tile, tiles;                 // tokens, tokens per tile (a multiple of kSortThreads)
  int shift, bits;
  int first;
  int* error_word;
};

// Element i of a pass's input.  The first pass makes the pairs: a token's word, or `vocab` (behind every word) for padding
// and for indices outside the table.  The others read what other blocks wrote: past the L1 cache.
__device__ __forceinline__ uint2 sort_pair(const SortPass& p, int i) {
  if (!p.first) return __ldcg(p.in + i);
  const int id = load_index(p.indices, p.index_type, i, p.vocab);
  if (id < 0) atomicOr(p.error_word, kErrorTokenIndex);
  return make_uint2(static_cast<unsigned>((id < 0 || id == p.padding) ? p.vocab : id), static_cast<unsigned>(i));
}

// The words that a block's tokens name, gathered in shared memory (a frequent word asks for its bit thousands of times) and
// handed over once, where the vocabulary's bits fit; by themselves, and only where the bit is not there yet, where not.
// (262144 tokens of 131072 words: the counting launch takes 44 us with an atomic a token, 7 so.)
constexpr int kPresentWords = 4096;                    // 131072 words: 16 KB
__device__ __forceinline__ void present_mark(const SortPass& p, unsigned* bits, unsigned word) {
  if (word >= static_cast<unsigned>(p.vocab)) return;
  const unsigned bit = 1u << (word & 31);
  if (p.vocab <= 32 * kPresentWords) {
    if (!(bits[word >> 5] & bit)) atomicOr(bits + (word >> 5), bit);
  } else if (!(__ldcg(p.present + (word >> 5)) & bit)) {
    atomicOr(p.present + (word >> 5), bit);
  }
}
__device__ __forceinline__ void present_clear(const SortPass& p, unsigned* bits) {
  if (p.vocab <= 32 * kPresentWords)
    for (int i = threadIdx.x; i <= (p.vocab - 1) >> 5; i += kSortThreads) bits[i] = 0;
}
__device__ __forceinline__ void present_hand_over(const SortPass& p, const unsigned* bits) {
  if (p.vocab <= 32 * kPresentWords)
    for (int i = threadIdx.x; i <= (p.vocab - 1) >> 5; i += kSortThreads)
      if (bits[i]) atomicOr(p.present + i, bits[i]);
}

// A warp's strip of up to 32 * ITEMS tokens from `begin` on, in registers: token begin + 32 k + lane is item k.
template <int ITEMS>
__device__ __forceinline__ void sort_load(const SortPass& p, int begin, int end, uint2 (&item)[ITEMS]) {
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = begin + 32 * k + (threadIdx.x & 31);
    if (i < end) item[k] = sort_pair(p, i);
  }
}
// Counts the strip's digits in the warp's own counters (zeroed) and gives every item its rank among the items of its digit
// that come before it in the strip: 32 at a time, lanes with the same digit in lane order.
template <int ITEMS>
__device__ __forceinline__ void sort_rank(const SortPass& p, int begin, int end, const uint2 (&item)[ITEMS], unsigned* hist, unsigned (&rank)[ITEMS]) {
  const int lane = threadIdx.x & 31;
  const unsigned mask = (1u << p.bits) - 1;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    if (begin + 32 * k >= end) break;                  // the same for the whole warp
    const bool live = begin + 32 * k + lane < end;
    const unsigned digit = live ? (item[k].x >> p.shift) & mask : 0xffffffffu;
    const unsigned peers = __match_any_sync(0xffffffffu, digit);
    const unsigned ahead = __popc(peers & ((1u << lane) - 1));
    if (live) rank[k] = hist[digit] + ahead;
    __syncwarp();
    if (live && ahead == 0) hist[digit] += __popc(peers);
    __syncwarp();
  }
}
// Writes the items to their places: offset[digit] is where the strip's first item with that digit goes.
template <int ITEMS>
__device__ __forceinline__ void sort_place(const SortPass& p, int begin, int end, const uint2 (&item)[ITEMS], const unsigned* offset, const unsigned (&rank)[ITEMS]) {
  const unsigned mask = (1u << p.bits) - 1;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
    if (begin + 32 * k + static_cast<int>(threadIdx.x & 31) < end) p.out[offset[(item[k].x >> p.shift) & mask] + rank[k]] = item[k];
}

// Exclusive prefix sum over the kSortThreads threads of a block.
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned* warp_sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  unsigned before = lane < warp ? warp_sums[lane & (kSortWarps - 1)] : 0;
  before = __reduce_add_sync(0xffffffffu, before);
  __syncthreads();
  return before + x - v;
}
// The warps' counts of digit d become the places of their first items, from `base` on; returns the digit's total.
__device__ __forceinline__ unsigned sort_total(const unsigned* smem, int bins, int d) {
  unsigned sum = 0;
#pragma unroll
  for (int k = 0; k < kSortWarps; ++k) sum += smem[k * bins + d];
  return sum;
}
__device__ __forceinline__ void sort_offsets(unsigned* smem, int bins, int d, unsigned base) {
  unsigned c[kSortWarps];
#pragma unroll
  for (int k = 0; k < kSortWarps; ++k) c[k] = smem[k * bins + d];
#pragma unroll
  for (int k = 0; k < kSortWarps; ++k) { smem[k * bins + d] = base; base += c[k]; }
}

// The sort of many tokens, three launches a digit.  Counts of every tile:
static __global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const SortPass p) {
  pdl_prologue();
  constexpr int ITEMS = kSortTile / kSortThreads;
  __shared__ unsigned hist[kSortMaxBins];
  __shared__ unsigned bits[kPresentWords];
  const int bins = 1 << p.bits, d = threadIdx.x;
  const bool note = p.first && p.present;
  if (d < bins) hist[d] = 0;
  if (note) present_clear(p, bits);
  if (p.first && blockIdx.x == 0 && d == 0) *p.crossing = 0;
  uint2 item[ITEMS];
  const int begin = blockIdx.x * p.tile + (d >> 5) * (32 * ITEMS), end = min(p.n, begin + 32 * ITEMS);
  sort_load<ITEMS>(p, begin, end, item);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
    if (begin + 32 * k + (d & 31) < end) {
      atomicAdd(&hist[(item[k].x >> p.shift) & (bins - 1)], 1u);
      if (note) present_mark(p, bits, item[k].x);
    }
  __syncthreads();
  if (d < bins) p.counts[static_cast<size_t>(d) * p.tiles + blockIdx.x] = hist[d];
  if (note) present_hand_over(p, bits);
}

// Exclusive prefix of a bin's counts over the tiles, and its total: one warp per bin.
static __global__ void __launch_bounds__(256)
sort_prefix_kernel(const SortPass p) {
  pdl_prologue();
  const int bin = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (bin >= (1 << p.bits)) return;
  unsigned* c = p.counts + static_cast<size_t>(bin) * p.tiles;
  unsigned run = 0;
  for (int b = 0; b < p.tiles; b += 32) {
    const unsigned v = b + lane < p.tiles ? c[b + lane] : 0;
    unsigned x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    if (b + lane < p.tiles) c[b + lane] = run + x - v;
    run += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) p.totals[bin] = run;
}

static __global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(const SortPass p, const ZeroRows z) {
  pdl_prologue();
  if (blockIdx.x >= p.tiles) {
    zero_words(z, (blockIdx.x - p.tiles) * static_cast<long long>(kSortWarps) + (threadIdx.x >> 5), (gridDim.x - p.tiles) * static_cast<long long>(kSortWarps));
    return;
  }
  constexpr int ITEMS = kSortTile / kSortThreads;
  extern __shared__ unsigned sort_smem[];              // [warps][bins]
  __shared__ unsigned warp_sums[kSortWarps];
  const int bins = 1 << p.bits, warp = threadIdx.x >> 5, d = threadIdx.x;     // bins <= kSortThreads: a thread per bin
  uint2 item[ITEMS];
  unsigned rank[ITEMS];
  const int begin = blockIdx.x * p.tile + warp * (32 * ITEMS), end = min(p.n, begin + 32 * ITEMS);
  sort_load<ITEMS>(p, begin, end, item);
  const unsigned before = d < bins ? p.counts[static_cast<size_t>(d) * p.tiles + blockIdx.x] : 0;
  const unsigned base = block_exclusive(d < bins ? p.totals[d] : 0, warp_sums) + before;
  for (int i = d; i < bins * kSortWarps; i += kSortThreads) sort_smem[i] = 0;
  __syncthreads();
  sort_rank<ITEMS>(p, begin, end, item, sort_smem + warp * bins, rank);
  __syncthreads();
  if (d < bins) sort_offsets(sort_smem, bins, d, base);
  __syncthreads();
  sort_place<ITEMS>(p, begin, end, item, sort_smem + warp * bins, rank);
}

// The whole sort as one launch: one block, or a cluster of eight with a tile each.  Per pass every block ranks the items
// of its warps' strips, the blocks read each other's counts through distributed shared memory, and the pairs go to their
// places in the blocks' shared memory, the last pass's to global memory.  The other clusters of the launch clear the
// gradient meanwhile, all of it: the rows that are summed later are few here (at most a row a token), and waiting for the
// list of those that are not would cost more than writing them twice.  Bound by the latency of its barriers: 8 us for 4999
// tokens, hidden behind the clearing of a table of 134 MB (20 us).
constexpr int kSortCluster = 8;
constexpr int kSortClusterTile = kSortClusterTokens / kSortCluster;
struct SortAll {
  SortPass pass;                      // tile: a power of two, 2^tile_shift
  int tile_shift;
  uint2* out;
  int passes;
  float* clear;                       // [zeros] floats that are set to zero
  long long zeros;
};
static __global__ void __launch_bounds__(kSortThreads)
sort_cluster_kernel(const SortAll all) {
  pdl_prologue();
  constexpr int ITEMS = kSortClusterTile / kSortThreads;
  extern __shared__ uint2 sort_pairs[];                // [tile] pairs, then [warps][bins] counters
  __shared__ unsigned counts[kSortMaxBins];            // of this block, read by the others
  __shared__ unsigned warp_sums[kSortWarps];
  SortPass p = all.pass;
  unsigned* const hist = reinterpret_cast<unsigned*>(sort_pairs + p.tile);
  const int bins = 1 << p.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x, here = blockIdx.x, blocks = p.tiles;
  if (here >= blocks) {
    fill_zero(all.zeros, all.clear, (here - blocks) * static_cast<long long>(kSortThreads) + d, (gridDim.x - blocks) * static_cast<long long>(kSortThreads));
    return;
  }
  const int strip = p.tile / kSortWarps;
  const int begin = min(p.n, here * p.tile + warp * strip), end = min(p.n, begin + strip);
  if (here == 0 && d == 0) *p.crossing = 0;
  const unsigned mask = bins - 1, tile_mask = p.tile - 1, mine = smem_u32(sort_pairs);
  uint2 item[ITEMS];
  unsigned rank[ITEMS];
  for (int pass = 0; pass < all.passes; ++pass) {
    p.first = pass == 0;
    p.shift = pass * p.bits;
    if (p.first) {
      sort_load<ITEMS>(p, begin, end, item);
    } else {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (begin + 32 * k + lane < end) item[k] = sort_pairs[(begin + 32 * k + lane) & tile_mask];
    }
    for (int i = d; i < bins * kSortWarps; i += kSortThreads) hist[i] = 0;
    __syncthreads();
    sort_rank<ITEMS>(p, begin, end, item, hist + warp * bins, rank);
    __syncthreads();
    unsigned before = 0, total = 0;
    if (d < bins) total = counts[d] = sort_total(hist, bins, d);
    if (blocks > 1) {
      cluster_sync_all();                              // (and every block has its pairs in registers)
      if (d < bins) {
        unsigned v[kSortCluster];
#pragma unroll
        for (int r = 0; r < kSortCluster; ++r)
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(map_to_cta(smem_u32(counts + d), r)) : "memory");
        total = 0;
#pragma unroll
        for (int r = 0; r < kSortCluster; ++r) {
          if (r < here) before += v[r];
          total += v[r];
        }
      }
    }
    const unsigned base = block_exclusive(total, warp_sums) + before;
    if (d < bins) sort_offsets(hist, bins, d, base);
    __syncthreads();
    if (pass + 1 == all.passes) {
      p.out = all.out;
      sort_place<ITEMS>(p, begin, end, item, hist + warp * bins, rank);
    } else {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
        if (begin + 32 * k + lane < end) {
          const unsigned to = hist[warp * bins + ((item[k].x >> p.shift) & mask)] + rank[k];
          const unsigned at = map_to_cta(mine + 8 * (to & tile_mask), to >> all.tile_shift);
          asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(item[k].x), "r"(item[k].y) : "memory");
        }
    }
    cluster_sync_all();                                // the pairs are in place, and no block's memory is still being used by others
  }
}

// ---------------------------------------------------------------- sums over the sorted tokens
struct WordSums {
  const uint2* pairs;                 // (word, token), sorted
  unsigned* crossing;                 // how many words cross a border between chunks, and the chunks in which they begin
  unsigned* crossing_chunk;
  int n, vocab, dim, chunk, chunks, slabs;
  float scale;
  int accumulate;
  const float* dy;
  float* dtable;
  float* partial;                     // [chunks][2][dim]: of the word that enters the chunk, of the one that leaves it
};
__device__ __forceinline__ void add4(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }

template <int VEC>
__device__ __forceinline__ void store_word(const WordSums& p, unsigned word, int slab, int lane, float4 sum, const float4& old) {
  sum.x = fmaf(p.scale, sum.x, old.x); sum.y = fmaf(p.scale, sum.y, old.y); sum.z = fmaf(p.scale, sum.z, old.z); sum.w = fmaf(p.scale, sum.w, old.w);
  store_cols<VEC>(p.dtable + static_cast<long long>(word) * p.dim, slab, lane, p.dim, sum);
}

// A warp a chunk and slab.  U rows are in flight per lane; with ACCUMULATE the row that a word's sum is added to is fetched
// with the word's first row, not when the sum is done (in a long tail of words that occur once that would be one memory
// latency a row).  Bound by memory on a long batch: 262144 rows of 1024 take 200 us (1.2 GB at 6.1 TB/s); by its waves of
// blocks on a short one (16384 rows: 16 to 18 us for 97 MB, at four blocks a SM; 22 at three).
template <int VEC, bool ACCUMULATE>
static __global__ void __launch_bounds__(256, VEC == 4 && !ACCUMULATE ? 4 : 2)
word_sums_kernel(const WordSums p) {
  pdl_prologue();
  constexpr int U = 8;
  const int lane = threadIdx.x & 31;
  const long long id = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int chunk = static_cast<int>(id / p.slabs), slab = static_cast<int>(id % p.slabs);
  if (chunk >= p.chunks) return;
  const int begin = chunk * p.chunk, end = min(p.n, begin + p.chunk);
  const unsigned none = 0xffffffffu, dropped = static_cast<unsigned>(p.vocab);
  const unsigned before = begin > 0 ? p.pairs[begin - 1].x : none, after = end < p.n ? p.pairs[end].x : none;
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float4 sum = zero, old = zero;
  unsigned word = p.pairs[begin].x;
  bool entered = word == before;                       // the word began in an earlier chunk
  if (ACCUMULATE && !entered && word < dropped) old = load_cols<VEC>(p.dtable + static_cast<long long>(word) * p.dim, slab, lane, p.dim);
  for (int b = begin; b < end; b += 32) {
    const int count = min(32, end - b);
    const uint2 pair = lane < count ? p.pairs[b + lane] : make_uint2(none, 0);
    for (int j = 0; j < count; j += U) {
      // lanes behind the count hold `none`; j + u stays below 32 because the count is at most that and U divides 32
      float4 v[U], o[ACCUMULATE ? U : 1];
      unsigned last = word;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned k = __shfl_sync(0xffffffffu, pair.x, j + u), t = __shfl_sync(0xffffffffu, pair.y, j + u);
        v[u] = k < dropped ? load_cols<VEC>(p.dy + static_cast<long long>(t) * p.dim, slab, lane, p.dim) : zero;
        if (ACCUMULATE) {
          o[u] = k < dropped && k != last ? load_cols<VEC>(p.dtable + static_cast<long long>(k) * p.dim, slab, lane, p.dim) : zero;
          last = k;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned k = __shfl_sync(0xffffffffu, pair.x, j + u);
        if (k == none) break;
        if (k != word) {                               // the word ends here
          if (word < dropped) {
            if (entered) store_cols<VEC>(p.partial + (2LL * chunk) * p.dim, slab, lane, p.dim, sum);
            else store_word<VEC>(p, word, slab, lane, sum, old);
          }
          word = k;
          entered = false;
          sum = zero;
          if (ACCUMULATE) old = o[u];
        }
        add4(sum, v[u]);
      }
    }
  }
  if (word >= dropped) return;
  if (entered) {
    store_cols<VEC>(p.partial + (2LL * chunk) * p.dim, slab, lane, p.dim, sum);
  } else if (word == after) {
    store_cols<VEC>(p.partial + (2LL * chunk + 1) * p.dim, slab, lane, p.dim, sum);
    if (slab == 0 && lane == 0) p.crossing_chunk[atomicAdd(p.crossing, 1u)] = static_cast<unsigned>(chunk);
  } else {
    store_word<VEC>(p, word, slab, lane, sum, old);
  }
}

// The words that cross chunks.  (The order of the list does not matter: each entry is a word of its own.)  A warp takes a
// slab of a word and adds its partial sums in chunk order; where there are many, the block's eight warps add up eight runs
// of them, and their sums are added in order.  Bound by latency: 10 us for the 1300 words that cross in 262144 tokens (33 us
// with a block a word, whose neighbours in the list were slabs of the same word).
template <int VEC>
static __global__ void __launch_bounds__(256)
word_join_kernel(const WordSums p) {
  pdl_prologue();
  constexpr int U = 8, MANY = 32;
  __shared__ float4 run_sums[8][32];
  __shared__ int many_last[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add_run = [&](int chunk, int slab, int from, int to) {   // partial sums [from, to) of the word that begins in `chunk`
    float4 sum = zero;
    for (int j = from; j < to; j += U) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = j + u < to ? load_cols<VEC>(p.partial + (2LL * (j + u) + (j + u == chunk)) * p.dim, slab, lane, p.dim) : zero;
#pragma unroll
      for (int u = 0; u < U; ++u) add4(sum, v[u]);
    }
    return sum;
  };
  auto finish = [&](unsigned word, int slab, const float4& sum) {
    store_word<VEC>(p, word, slab, lane, sum, p.accumulate ? load_cols<VEC>(p.dtable + static_cast<long long>(word) * p.dim, slab, lane, p.dim) : zero);
  };
  const long long items = static_cast<long long>(*p.crossing) * p.slabs;
  // neighbours in the list (the slabs of one word) go to different blocks, so that a frequent word keeps many of them busy
  for (long long first = blockIdx.x; first < items; first += gridDim.x * 8LL) {
    const long long item = first + static_cast<long long>(warp) * gridDim.x;
    int last = -1;
    if (item < items) {
      const int chunk = static_cast<int>(p.crossing_chunk[item / p.slabs]), slab = static_cast<int>(item % p.slabs);
      // most words reach one chunk behind their first: what depends on the chunk alone is fetched together
      const unsigned word = p.pairs[(chunk + 1LL) * p.chunk].x;
      const float4 begun = load_cols<VEC>(p.partial + (2LL * chunk + 1) * p.dim, slab, lane, p.dim);
      const float4 behind = load_cols<VEC>(p.partial + (2LL * chunk + 2) * p.dim, slab, lane, p.dim);
      last = chunk + 1;                                 // the last chunk that the word reaches
      for (;;) {
        const long long border = static_cast<long long>(last + lane + 1) * p.chunk;       // first token of the chunk behind it
        const bool on = border < p.n && p.pairs[border].x == word;
        const unsigned stops = __ballot_sync(0xffffffffu, !on);
        if (stops) { last += __ffs(stops) - 1; break; }
        last += 32;
      }
      if (last - chunk < MANY) {
        float4 sum = begun;
        add4(sum, behind);
        if (last > chunk + 1) add4(sum, add_run(chunk, slab, chunk + 2, last + 1));
        finish(word, slab, sum);
        last = -1;
      }
    }
    if (lane == 0) many_last[warp] = last;
    __syncthreads();
    for (int k = 0; k < 8; ++k) {
      const int to = many_last[k];
      if (to < 0) continue;                             // the same for the whole block
      const long long which = first + static_cast<long long>(k) * gridDim.x;
      const int chunk = static_cast<int>(p.crossing_chunk[which / p.slabs]), slab = static_cast<int>(which % p.slabs);
      const int run = (to - chunk + 8) / 8, from = chunk + warp * run;
      float4 sum = add_run(chunk, slab, from, min(to + 1, from + run));
      run_sums[warp][lane] = sum;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int o = 1; o < 8; ++o) add4(sum, run_sums[o][lane]);
        finish(p.pairs[(chunk + 1LL) * p.chunk].x, slab, sum);
      }
      __syncthreads();
    }
    __syncthreads();                                    // many_last has been read
  }
}

}  // namespace snb
