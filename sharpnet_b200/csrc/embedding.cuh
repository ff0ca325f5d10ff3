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
// other with their loads in flight together.
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

// ---------------------------------------------------------------- stable sort of (word, token), one digit a pass
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxBits = 9;                      // digit of at most 9 bits: 16 warps x 512 counters = 32 KB
constexpr int kSortMaxBins = 1 << kSortMaxBits;

struct SortPass {
  const void* indices;                // the caller's indices: read by the first pass in place of `in`
  int index_type, vocab, padding;
  const uint2* in;                    // (word, token)
  uint2* out;
  unsigned *counts;                   // [bins][tiles]
  unsigned *totals;                   // [bins]
  unsigned *present;                  // a bit per word that occurs, or NULL
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
  return make_uint2(static_cast<unsigned>((id < 0 || id == p.padding) ? p.vocab : id), static_cast<unsigned>(i));
}
// What the first pass notes down about token i besides.
__device__ __forceinline__ void sort_note(const SortPass& p, int i, unsigned word) {
  if (load_index(p.indices, p.index_type, i, p.vocab) < 0) atomicOr(p.error_word, kErrorTokenIndex);
  if (p.present && word < static_cast<unsigned>(p.vocab)) {
    const unsigned bit = 1u << (word & 31);
    if (!(__ldcg(p.present + (word >> 5)) & bit)) atomicOr(p.present + (word >> 5), bit);     // frequent words ask once
  }
}

static __global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const SortPass p) {
  pdl_prologue();
  __shared__ unsigned hist[kSortMaxBins];
  const int bins = 1 << p.bits;
  for (int d = threadIdx.x; d < bins; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const int begin = blockIdx.x * p.tile, end = min(p.n, begin + p.tile);
  for (int i = begin + threadIdx.x; i < end; i += kSortThreads) {
    const unsigned word = sort_pair(p, i).x;
    if (p.first) sort_note(p, i, word);
    atomicAdd(&hist[(word >> p.shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) p.counts[static_cast<size_t>(d) * p.tiles + blockIdx.x] = hist[d];
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
  unsigned before = 0;
  for (int k = 0; k < warp; ++k) before += warp_sums[k];
  __syncthreads();
  return before + x - v;
}

// Counts the digits of one warp's strip [begin, end) into hist (one counter per bin, the warp's own, zeroed); with NOTE
// the first pass notes its tokens down.
template <bool NOTE>
__device__ __forceinline__ void sort_strip_count(const SortPass& p, int begin, int end, unsigned* hist) {
  const int lane = threadIdx.x & 31;
  const unsigned mask = (1u << p.bits) - 1;
  for (int i = begin + lane; i < end; i += 32) {
    const unsigned word = sort_pair(p, i).x;
    if (NOTE && p.first) sort_note(p, i, word);
    atomicAdd(&hist[(word >> p.shift) & mask], 1u);
  }
}
// Writes the pairs of the strip to their places: offset[digit] is where the strip's first pair with that digit goes.
// Tokens are taken 32 at a time in order; lanes with the same digit take consecutive places in lane order.
__device__ __forceinline__ void sort_strip_place(const SortPass& p, int begin, int end, unsigned* offset) {
  const int lane = threadIdx.x & 31;
  const unsigned mask = (1u << p.bits) - 1;
  for (int b = begin; b < end; b += 32) {
    const int i = b + lane;
    const bool live = i < end;
    const uint2 pair = live ? sort_pair(p, i) : make_uint2(0, 0);
    const unsigned digit = live ? (pair.x >> p.shift) & mask : 0xffffffffu;
    const unsigned peers = __match_any_sync(0xffffffffu, digit);
    const unsigned rank = __popc(peers & ((1u << lane) - 1));
    unsigned to = 0;
    if (live) to = offset[digit] + rank;
    __syncwarp();
    if (live && rank == 0) offset[digit] += __popc(peers);
    __syncwarp();
    if (live) p.out[to] = pair;
  }
}

static __global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(const SortPass p) {
  pdl_prologue();
  extern __shared__ unsigned sort_smem[];              // [warps][bins]
  __shared__ unsigned warp_sums[kSortWarps];
  const int bins = 1 << p.bits, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < bins * kSortWarps; d += kSortThreads) sort_smem[d] = 0;
  __syncthreads();
  const int strip = p.tile / kSortWarps;
  const int begin = min(p.n, blockIdx.x * p.tile + warp * strip);
  const int end = min(p.n, begin + strip);
  sort_strip_count<false>(p, begin, end, sort_smem + warp * bins);
  __syncthreads();
  const int d = threadIdx.x;                           // bins <= kSortThreads: a thread per bin
  unsigned base = block_exclusive(d < bins ? p.totals[d] : 0, warp_sums);
  if (d < bins) {
    base += p.counts[static_cast<size_t>(d) * p.tiles + blockIdx.x];
    for (int k = 0; k < kSortWarps; ++k) {
      const unsigned c = sort_smem[k * bins + d];
      sort_smem[k * bins + d] = base;
      base += c;
    }
  }
  __syncthreads();
  sort_strip_place(p, begin, end, sort_smem + warp * bins);
}

// The whole sort as one launch for up to 32768 tokens: one block, or a cluster of eight with a tile each.  Per pass every
// block counts the digits of its warps' strips, the blocks read each other's counts through distributed shared memory,
// and the pairs go to their places in global memory, which the barrier at the end of a pass makes visible to the cluster.
// Three launches a digit cost what a small batch costs altogether (4999 tokens: 27 -> 12 us with the sums).
constexpr int kSortClusterTokens = 32768;
struct SortAll {
  SortPass pass;
  uint2 *buffer[2];
  int passes;
};
static __global__ void __launch_bounds__(kSortThreads)
sort_cluster_kernel(const SortAll all) {
  pdl_prologue();
  extern __shared__ unsigned sort_smem[];              // [warps][bins]
  __shared__ unsigned counts[kSortMaxBins];            // of this block, read by the others
  __shared__ unsigned warp_sums[kSortWarps];
  SortPass p = all.pass;
  const int bins = 1 << p.bits, warp = threadIdx.x >> 5, d = threadIdx.x, rank = blockIdx.x, blocks = gridDim.x;
  const int strip = p.tile / kSortWarps;
  const int begin = min(p.n, rank * p.tile + warp * strip), end = min(p.n, begin + strip);
  if (p.present) {
    for (int i = rank * kSortThreads + d; i <= (p.vocab - 1) >> 5; i += blocks * kSortThreads) p.present[i] = 0;
    cluster_sync_all();
  }
  for (int pass = 0; pass < all.passes; ++pass) {
    p.first = pass == 0;
    p.shift = pass * p.bits;
    p.in = all.buffer[(pass + 1) & 1];
    p.out = all.buffer[pass & 1];
    for (int i = d; i < bins * kSortWarps; i += kSortThreads) sort_smem[i] = 0;
    __syncthreads();
    sort_strip_count<true>(p, begin, end, sort_smem + warp * bins);
    __syncthreads();
    unsigned sum = 0;
    if (d < bins) {
      for (int k = 0; k < kSortWarps; ++k) sum += sort_smem[k * bins + d];
      counts[d] = sum;
    }
    cluster_sync_all();
    unsigned before = 0, total = 0;
    if (d < bins) {
      for (int r = 0; r < blocks; ++r) {
        unsigned v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(smem_u32(counts + d), r)) : "memory");
        if (r < rank) before += v;
        total += v;
      }
    }
    unsigned base = block_exclusive(total, warp_sums) + before;
    if (d < bins) {
      for (int k = 0; k < kSortWarps; ++k) {
        const unsigned c = sort_smem[k * bins + d];
        sort_smem[k * bins + d] = base;
        base += c;
      }
    }
    __syncthreads();
    sort_strip_place(p, begin, end, sort_smem + warp * bins);
    cluster_sync_all();
  }
}

// ---------------------------------------------------------------- sums over the sorted tokens
static __global__ void __launch_bounds__(256)
fill_zero_kernel(long long n, float* __restrict__ p) {
  pdl_prologue();
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long tid = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  const long long head = min(n, static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) >> 2);
  const long long quads = (n - head) >> 2;
  for (long long i = tid; i < quads; i += stride) reinterpret_cast<float4*>(p + head)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (tid < head) p[tid] = 0.0f;
  if (head + 4 * quads + tid < n) p[head + 4 * quads + tid] = 0.0f;
}

struct WordSums {
  const uint2* pairs;                 // (word, token), sorted
  const unsigned* present;            // a bit per word that occurs; NULL: rows of other words are left as they are
  int n, vocab, dim, chunk, chunks, slabs;
  long long sum_blocks;               // blocks that add rows; the others write the rows of words that do not occur
  float scale;
  int accumulate;
  const float* dy;
  float* dtable;
  float* partial;                     // [chunks][2][dim]: of the word that enters the chunk, of the one that leaves it
};
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
__device__ __forceinline__ void add4(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }

template <int VEC>
__device__ __forceinline__ void store_word(const WordSums& p, unsigned word, int slab, int lane, float4 sum) {
  float* row = p.dtable + static_cast<long long>(word) * p.dim;
  sum.x *= p.scale; sum.y *= p.scale; sum.z *= p.scale; sum.w *= p.scale;
  if (p.accumulate) add4(sum, load_cols<VEC>(row, slab, lane, p.dim));
  store_cols<VEC>(row, slab, lane, p.dim, sum);
}

// A slab of the rows of 32 words: zeros where the word does not occur.
template <int VEC>
__device__ __forceinline__ void zero_words(const WordSums& p, long long id, int lane) {
  const long long group = id / p.slabs;
  const int slab = static_cast<int>(id % p.slabs);
  const long long first = 32 * group;
  if (first >= p.vocab) return;
  const unsigned present = p.present[group];
  const int words = static_cast<int>(min(32LL, p.vocab - first));
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (VEC == 4 && p.dim < kSlab) {                     // narrow rows: as many side by side as a warp's width holds
    const int quads = p.dim >> 2;
    for (int i = lane; i < words * quads; i += 32) {
      const int w = i / quads;
      if (!(present >> w & 1)) reinterpret_cast<float4*>(p.dtable + first * p.dim)[i] = zero;
    }
    return;
  }
  for (int w = 0; w < words; ++w)
    if (!(present >> w & 1)) store_cols<VEC>(p.dtable + (first + w) * p.dim, slab, lane, p.dim, zero);
}

template <int VEC>
static __global__ void __launch_bounds__(256)
word_sums_kernel(const WordSums p) {
  pdl_prologue();
  constexpr int U = 8;                                 // rows in flight per lane
  const int lane = threadIdx.x & 31;
  if (blockIdx.x >= p.sum_blocks) {
    zero_words<VEC>(p, (blockIdx.x - p.sum_blocks) * 8LL + (threadIdx.x >> 5), lane);
    return;
  }
  const long long id = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int chunk = static_cast<int>(id / p.slabs), slab = static_cast<int>(id % p.slabs);
  if (chunk >= p.chunks) return;
  const int begin = chunk * p.chunk, end = min(p.n, begin + p.chunk);
  const unsigned none = 0xffffffffu, dropped = static_cast<unsigned>(p.vocab);
  const unsigned before = begin > 0 ? p.pairs[begin - 1].x : none, after = end < p.n ? p.pairs[end].x : none;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  unsigned word = p.pairs[begin].x;
  bool entered = word == before;                       // the word began in an earlier chunk
  for (int b = begin; b < end; b += 32) {
    const int count = min(32, end - b);
    const uint2 pair = lane < count ? p.pairs[b + lane] : make_uint2(none, 0);
    for (int j = 0; j < count; j += U) {
      float4 v[U];
      unsigned k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        k[u] = __shfl_sync(0xffffffffu, pair.x, (j + u) & 31);
        const unsigned t = __shfl_sync(0xffffffffu, pair.y, (j + u) & 31);
        if (j + u >= count) k[u] = none;
        v[u] = k[u] < dropped ? load_cols<VEC>(p.dy + static_cast<long long>(t) * p.dim, slab, lane, p.dim)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k[u] == none) continue;
        if (k[u] != word) {                            // the word ends here
          if (word < dropped) {
            if (entered) store_cols<VEC>(p.partial + (2LL * chunk) * p.dim, slab, lane, p.dim, sum);
            else store_word<VEC>(p, word, slab, lane, sum);
          }
          word = k[u];
          entered = false;
          sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        add4(sum, v[u]);
      }
    }
  }
  if (word >= dropped) return;
  if (entered) store_cols<VEC>(p.partial + (2LL * chunk) * p.dim, slab, lane, p.dim, sum);
  else if (word == after) store_cols<VEC>(p.partial + (2LL * chunk + 1) * p.dim, slab, lane, p.dim, sum);
  else store_word<VEC>(p, word, slab, lane, sum);
}

// The words that cross chunks: the warp of the chunk in which such a word begins adds its partial sums in chunk order.
template <int VEC>
static __global__ void __launch_bounds__(256)
word_join_kernel(const WordSums p) {
  pdl_prologue();
  constexpr int U = 8;
  const long long id = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int chunk = static_cast<int>(id / p.slabs), slab = static_cast<int>(id % p.slabs);
  if (chunk + 1 >= p.chunks) return;
  const int begin = chunk * p.chunk, end = begin + p.chunk;
  const unsigned word = p.pairs[end - 1].x;
  if (word >= static_cast<unsigned>(p.vocab) || p.pairs[end].x != word) return;          // nothing leaves this chunk
  if (begin > 0 && p.pairs[begin - 1].x == word) return;                                 // it began earlier
  // the last chunk that the word reaches
  int last = chunk + 1;
  for (;;) {
    const long long border = static_cast<long long>(last + lane + 1) * p.chunk;       // first token of the chunk behind it
    const bool on = border < p.n && p.pairs[border].x == word;
    const unsigned stops = __ballot_sync(0xffffffffu, !on);
    if (stops) { last += __ffs(stops) - 1; break; }
    last += 32;
  }
  float4 sum = load_cols<VEC>(p.partial + (2LL * chunk + 1) * p.dim, slab, lane, p.dim);
  for (int j = chunk + 1; j <= last; j += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = j + u <= last ? load_cols<VEC>(p.partial + 2LL * (j + u) * p.dim, slab, lane, p.dim) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u) add4(sum, v[u]);
  }
  store_word<VEC>(p, word, slab, lane, sum);
}

}  // namespace snb
