// Embedding lookup and its gradient.
//
//   lookup   out[i, :] = scale * table[token_i, :]                      (a row of zeros where the token is none)
//   gradient G[v, :] (+)= scale * sum over i with token_i = v of g[i, :]
//
// A token outside [0, vocab) - the usual -1 of padded positions - is no token: its row of the lookup is zero whatever the
// table holds, and it adds to nothing.
//
// The gradient is a keyed row sum with as many keys as the vocabulary has tokens, so the scheme of the keyed row
// sums (an accumulator row per key and work unit) does not carry over: here almost every key has no row at all or
// one, and a few have thousands. Up to kSmallMax positions one launch does it all (small_grad_kernel): a CTA per
// range of the table. Above that it runs as
//   1. a stable sort of the positions by token (counting ranks for short inputs, radix passes for long ones);
//   2. one pass over the rows in sorted order: fixed runs of kRun sorted rows, each summed by one group of threads
//      in fp32 registers, that finish every token that lies inside the run and leave one fp32 partial row for a
//      token that crosses either of its ends; the rows of the table that no token names are zeroed by further CTAs
//      of the same launch;
//   3. the partial rows of crossing tokens added up in order.
// The order of every addition is fixed by the positions alone: the result repeats bit for bit, without atomics on
// floating-point data.
#pragma once

#include "launch.cuh"
#include "vocab_common.cuh"

namespace raft_b200 {
namespace detail {
namespace emb {

// ---------------------------------------------------------------------------------------
// Lookup. A group of G lanes takes (row, segment of U * G vectors): U loads in flight per lane, neighbouring lanes on
// neighbouring vectors. Memory bound; nothing to reuse but rows that several tokens name, which L2 holds. U is four
// 16-byte vectors, sixteen narrow ones where rows lie off 16-byte boundaries (10007 x 1001 fp16:
// 16.3 us, 22.0 with four). 65536 x 4096 bf16: 120 us, 9.0 TB/s of rows read and written (L2 serves the repeated rows).
// ---------------------------------------------------------------------------------------
constexpr int kLookupThreads = 256;
template <typename T, int V>
constexpr int kLookupUnroll = V * int(sizeof(T)) >= 16 ? 4 : 16;

template <typename T, int V, typename TokT>
__global__ void __launch_bounds__(kLookupThreads)
lookup_kernel(T* out, int64_t ldo, const T* table, int64_t ldt, const TokT* tokens, int64_t n_tokens, int64_t n_cols,
              int64_t vocab, float scale, int lg, unsigned segs)
{
  grid_dep_sync();
  const int64_t gid = (int64_t(blockIdx.x) * kLookupThreads + threadIdx.x) >> lg;
  const int64_t row = gid / segs;
  const unsigned sg = unsigned(gid - row * segs);
  if (row >= n_tokens) return;
  const int G        = 1 << lg;
  const int lane     = int(threadIdx.x) & (G - 1);
  const int64_t tok  = int64_t(tokens[row]);
  const bool valid   = tok >= 0 && tok < vocab;
  const int64_t nvec = n_cols / V;
  const T* src       = table + (valid ? tok : 0) * ldt;
  T* dst             = out + row * ldo;
  constexpr int U    = kLookupUnroll<T, V>;
  const int64_t v0   = int64_t(sg) * (U << lg) + lane;
  Elems<T, V> r[U];
  // loads without conditions, so that all of them are under way at once: behind the row's end its last vector again, for
  // no token the table's first row
  if (vocab > 0 && nvec > 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + (int64_t(u) << lg);
      r[u].load(src + (v < nvec ? v : nvec - 1) * V);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + (int64_t(u) << lg);
    if (v < nvec) {
      float f[V];
      r[u].up(f);
#pragma unroll
      for (int i = 0; i < V; ++i)
        f[i] = valid ? f[i] * scale : 0.0f;
      r[u].down(f);
      r[u].store(dst + v * V);
    }
  }
  if constexpr (V > 1) {  // the columns behind the last whole vector
    const int64_t c = nvec * V + lane;
    if (sg == segs - 1) {
      for (int64_t j = c; j < n_cols; j += G)
        dst[j] = FloatIo<T>::down(valid ? FloatIo<T>::up(src[j]) * scale : 0.0f);
    }
  }
}

template <typename T, int V, typename TokT>
inline cudaError_t launch_lookup_v(T* out, int64_t ldo, const T* table, int64_t ldt, const TokT* tokens,
                                   int64_t n_tokens, int64_t n_cols, int64_t vocab, float scale, cudaStream_t stream)
{
  const int64_t nvec = n_cols / V > 0 ? n_cols / V : 1;
  const int64_t want = ceil_div<int64_t>(nvec, kLookupUnroll<T, V>);
  const int lg       = want >= 32 ? 5 : ilog2_floor(next_pow2(unsigned(want)));
  const int64_t segs = ceil_div<int64_t>(nvec, int64_t(kLookupUnroll<T, V>) << lg);
  if (segs > int64_t(0x7fffffff)) return cudaErrorInvalidValue;
  const int64_t per_cta = kLookupThreads >> lg;
  const int64_t max_row = int64_t(0x7fffffff) * per_cta / segs;  // rows of one launch
  for (int64_t r0 = 0; r0 < n_tokens; r0 += max_row) {
    const int64_t n = n_tokens - r0 < max_row ? n_tokens - r0 : max_row;
    (void)launch_dep(lookup_kernel<T, V, TokT>, dim3(unsigned(ceil_div<int64_t>(n * segs, per_cta))),
                     dim3(kLookupThreads), 0, stream, out + r0 * ldo, ldo, table, ldt, tokens + r0, n, n_cols, vocab,
                     scale, lg, unsigned(segs));
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, typename TokT>
inline cudaError_t launch_lookup(T* out, int64_t ldo, const T* table, int64_t ldt, const TokT* tokens,
                                 int64_t n_tokens, int64_t n_cols, int64_t vocab, float scale, cudaStream_t stream)
{
  if (n_tokens <= 0 || n_cols <= 0) return cudaSuccess;
  const int a = common_alignment({reinterpret_cast<uintptr_t>(out), reinterpret_cast<uintptr_t>(table),
                                  uintptr_t(ldo) * sizeof(T), uintptr_t(ldt) * sizeof(T)});
  constexpr int S = int(sizeof(T));
  if (a >= 16) return launch_lookup_v<T, 16 / S>(out, ldo, table, ldt, tokens, n_tokens, n_cols, vocab, scale, stream);
  if (a >= 4 && S < 4)
    return launch_lookup_v<T, (4 / S > 0 ? 4 / S : 1)>(out, ldo, table, ldt, tokens, n_tokens, n_cols, vocab, scale,
                                                       stream);
  return launch_lookup_v<T, 1>(out, ldo, table, ldt, tokens, n_tokens, n_cols, vocab, scale, stream);
}

// ---------------------------------------------------------------------------------------
// Sort of the positions by token. Keys are the tokens, `vocab` for "none" (sorted to the end).
// ---------------------------------------------------------------------------------------
template <typename TokT>
B2R_DI unsigned key_of(const TokT* tokens, int64_t i, unsigned vocab)
{
  const int64_t t = int64_t(tokens[i]);
  return t >= 0 && t < int64_t(vocab) ? unsigned(t) : vocab;
}

// Short inputs: the place of a position is the number of positions before it in (token, position) order. All keys
// sit in shared memory; kRankLanes lanes share the counting of one position. n^2 comparisons over the whole
// machine: below a few thousand positions that costs less than the launches of the radix passes.
constexpr int kRankThreads = 256;
constexpr int kRankLanes   = 8;
constexpr int kRankMax     = 8192;

template <typename TokT>
__global__ void __launch_bounds__(kRankThreads)
rank_sort_kernel(unsigned* skey, unsigned* spos, const TokT* tokens, int n, unsigned vocab)
{
  extern __shared__ unsigned keys[];
  grid_dep_sync();
  const int padded = (n + 4 * kRankLanes - 1) / (4 * kRankLanes) * (4 * kRankLanes);
  for (int i = int(threadIdx.x); i < padded; i += kRankThreads)
    keys[i] = i < n ? key_of(tokens, i, vocab) : 0xffffffffu;  // larger than any key, behind any position
  __syncthreads();
  const int lane      = int(threadIdx.x) & (kRankLanes - 1);
  const int me        = int(blockIdx.x) * (kRankThreads / kRankLanes) + int(threadIdx.x) / kRankLanes;
  const unsigned mine = me < n ? keys[me] : 0;
  int before          = 0;
  for (int j = lane * 4; j < padded; j += 4 * kRankLanes) {
    const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
    before += (k.x < mine || (k.x == mine && j < me)) ? 1 : 0;
    before += (k.y < mine || (k.y == mine && j + 1 < me)) ? 1 : 0;
    before += (k.z < mine || (k.z == mine && j + 2 < me)) ? 1 : 0;
    before += (k.w < mine || (k.w == mine && j + 3 < me)) ? 1 : 0;
  }
#pragma unroll
  for (int o = kRankLanes / 2; o > 0; o >>= 1)
    before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0 && me < n) {
    skey[before] = mine;
    spos[before] = unsigned(me);
  }
}

// Long inputs: least significant digit first, up to kRadixBits bits a pass. CTA b owns the contiguous tile b of
// the pass's input, warp w of it the contiguous part w of the tile. Per pass: digit counts per tile
// (radix_count_kernel for the first pass; the scatter of a pass counts for the next one on the way), then the
// scatter, which places digit d of tile b behind all smaller digits and behind digit d of the tiles before b, in
// the order of the input within (stable).
constexpr int kRadixBits    = 9;
constexpr int kRadixBins    = 1 << kRadixBits;
constexpr int kRadixThreads = 512;
constexpr int kRadixWarps   = kRadixThreads / 32;
constexpr int kRadixHeld    = 4;

// counts[tile][bin] of digit 0; zeroes `clear` (the counts of the next pass)
template <typename TokT>
__global__ void __launch_bounds__(kRadixThreads)
radix_count_kernel(unsigned* counts, unsigned* clear, const TokT* tokens, int64_t n, int64_t tile, unsigned vocab,
                   int bits)
{
  __shared__ unsigned hist[kRadixBins];
  grid_dep_sync();
  const int bins = 1 << bits;
  for (int d = int(threadIdx.x); d < bins; d += kRadixThreads) {
    hist[d]                              = 0;
    clear[size_t(blockIdx.x) * bins + d] = 0;
  }
  __syncthreads();
  const int64_t lo = int64_t(blockIdx.x) * tile;
  const int64_t hi = lo + tile < n ? lo + tile : n;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kRadixThreads)
    atomicAdd(&hist[key_of(tokens, i, vocab) & unsigned(bins - 1)], 1u);
  __syncthreads();
  for (int d = int(threadIdx.x); d < bins; d += kRadixThreads)
    counts[size_t(blockIdx.x) * bins + d] = hist[d];
}

// One scatter pass. `tokens` non-null: the first pass, keys come from the tokens and positions are 0, 1, ...
// `next` non-null: counts of the next pass's digit per tile of the output (integer atomics: order does not matter).
template <typename TokT>
__global__ void __launch_bounds__(kRadixThreads)
radix_scatter_kernel(unsigned* okey, unsigned* opos, const TokT* tokens, const unsigned* ikey, const unsigned* ipos,
                     const unsigned* counts, unsigned* next, int64_t n, int64_t tile, unsigned vocab, int shift,
                     int bits)
{
  __shared__ unsigned place[kRadixWarps][kRadixBins];  // per warp: first its digit counts, then its next places
  __shared__ unsigned warp_sum[kRadixWarps];
  grid_dep_sync();
  const int bins      = 1 << bits;
  const unsigned mask = unsigned(bins - 1);
  const int warp      = int(threadIdx.x) >> 5;
  const int lane      = int(threadIdx.x) & 31;
  for (int d = int(threadIdx.x); d < bins * kRadixWarps; d += kRadixThreads)
    place[d / bins][d % bins] = 0;
  __syncthreads();
  const int64_t lo   = int64_t(blockIdx.x) * tile;
  const int64_t hi   = lo + tile < n ? lo + tile : n;
  const int64_t part = (ceil_div<int64_t>(tile, kRadixWarps) + 31) / 32 * 32;
  int64_t wlo        = lo + int64_t(warp) * part;
  int64_t whi        = wlo + part < hi ? wlo + part : hi;
  // the warp's first kRadixHeld x 32 rows are kept in registers between counting and placing (all of them, in tiles of
  // up to 2048)
  unsigned held_k[kRadixHeld], held_p[kRadixHeld];
#pragma unroll
  for (int u = 0; u < kRadixHeld; ++u) {
    const int64_t i = wlo + u * 32 + lane;
    held_k[u] = held_p[u] = 0;
    if (i < whi) {
      held_k[u] = tokens != nullptr ? key_of(tokens, i, vocab) : ikey[i];
      held_p[u] = tokens != nullptr ? unsigned(i) : ipos[i];
    }
  }
#pragma unroll
  for (int u = 0; u < kRadixHeld; ++u)
    if (wlo + u * 32 + lane < whi) atomicAdd(&place[warp][(held_k[u] >> shift) & mask], 1u);
  for (int64_t i = wlo + kRadixHeld * 32 + lane; i < whi; i += 32) {
    const unsigned k = tokens != nullptr ? key_of(tokens, i, vocab) : ikey[i];
    atomicAdd(&place[warp][(k >> shift) & mask], 1u);
  }
  // thread d: rows of digit d in all tiles, and in the tiles before this one
  const int d     = int(threadIdx.x);
  unsigned before = 0, all = 0;
  if (d < bins) {
    const int tiles = int(gridDim.x);
    int b           = 0;
    for (; b + 8 <= tiles; b += 8) {
      unsigned c[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        c[u] = counts[size_t(b + u) * bins + d];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        all += c[u];
        before += b + u < int(blockIdx.x) ? c[u] : 0u;
      }
    }
    for (; b < tiles; ++b) {
      const unsigned c = counts[size_t(b) * bins + d];
      all += c;
      before += b < int(blockIdx.x) ? c : 0u;
    }
  }
  // exclusive scan of `all` over the digits (a digit per thread)
  unsigned incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  unsigned base = incl - all + before;
  for (int w = 0; w < warp; ++w)
    base += warp_sum[w];
  if (d < bins) {
#pragma unroll
    for (int w = 0; w < kRadixWarps; ++w) {
      const unsigned c = place[w][d];
      place[w][d]      = base;
      base += c;
    }
  }
  __syncthreads();
  const auto put = [&](bool on, unsigned k, unsigned p) {
    const unsigned dig  = on ? (k >> shift) & mask : 0xffffffffu;  // lanes without a row match each other only
    const unsigned same = __match_any_sync(0xffffffffu, dig);
    const int rank      = __popc(same & ((1u << lane) - 1u));
    unsigned at         = 0;
    if (on) at = place[warp][dig] + unsigned(rank);
    __syncwarp();
    if (on && rank == 0) place[warp][dig] += unsigned(__popc(same));
    __syncwarp();
    if (on) {
      okey[at] = k;
      opos[at] = p;
      if (next != nullptr) atomicAdd(&next[size_t(at / tile) * bins + ((k >> (shift + bits)) & mask)], 1u);
    }
  };
#pragma unroll
  for (int u = 0; u < kRadixHeld; ++u)
    put(wlo + u * 32 + lane < whi, held_k[u], held_p[u]);
  for (int64_t i0 = wlo + kRadixHeld * 32; i0 < whi; i0 += 32) {
    const int64_t i  = i0 + lane;
    const bool on    = i < whi;
    const unsigned k = !on ? 0u : (tokens != nullptr ? key_of(tokens, i, vocab) : ikey[i]);
    const unsigned p = !on ? 0u : (tokens != nullptr ? unsigned(i) : ipos[i]);
    put(on, k, p);
  }
}

// ---------------------------------------------------------------------------------------
// The pass over the rows.
// ---------------------------------------------------------------------------------------
constexpr int kSumThreads = 128;
constexpr int kSumBatch   = 8;  // rows a thread has in flight

// old + scale * acc, rounded once to the output's type
template <typename OutT, int V>
B2R_DI void store_sum(OutT* dst, const float (&acc)[V], float scale, bool accumulate)
{
  Elems<OutT, V> o;
  float f[V];
  if (accumulate) {
    o.load(dst);
    o.up(f);
#pragma unroll
    for (int i = 0; i < V; ++i)
      f[i] = fmaf(acc[i], scale, f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      f[i] = acc[i] * scale;
  }
  o.down(f);
  o.store(dst);
}

// V fp32 partial sums to or from scratch (16-byte aligned for V = 4, 8)
template <int V>
B2R_DI void store_partial(float* dst, const float (&acc)[V])
{
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int q = 0; q < V / W; ++q) {
    VecOf<float, W> o;
#pragma unroll
    for (int i = 0; i < W; ++i)
      o.e[i] = acc[q * W + i];
    reinterpret_cast<VecOf<float, W>*>(dst)[q] = o;
  }
}
template <int V>
B2R_DI void load_partial(float (&acc)[V], const float* src)
{
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int q = 0; q < V / W; ++q) {
    const VecOf<float, W> o = reinterpret_cast<const VecOf<float, W>*>(src)[q];
#pragma unroll
    for (int i = 0; i < W; ++i)
      acc[q * W + i] = o.e[i];
  }
}

// Zeroes a row, `threads` threads of which this is `lane`: 16-byte stores between the row's 16-byte boundaries.
template <typename T>
B2R_DI void zero_row(T* row, int64_t n_cols, int lane, int threads)
{
  const int64_t ahead = int64_t((16 - int(uintptr_t(row) & 15u)) & 15) / int64_t(sizeof(T));
  const int64_t head  = ahead < n_cols ? ahead : n_cols;
  const int64_t whole = (n_cols - head) / (16 / int64_t(sizeof(T)));
  const int64_t tail  = head + whole * (16 / int64_t(sizeof(T)));
  for (int64_t j = lane; j < whole; j += threads)
    reinterpret_cast<uint4*>(row + head)[j] = make_uint4(0, 0, 0, 0);
  for (int64_t j = lane; j < head; j += threads)
    row[j] = FloatIo<T>::down(0.0f);
  for (int64_t j = tail + lane; j < n_cols; j += threads)
    row[j] = FloatIo<T>::down(0.0f);
}

constexpr int kFold = 8;

struct SumShape {
  int lg;          // log2 of the threads of a group
  unsigned slabs;  // column slabs of U x (1 << lg) vectors
  int run;         // sorted rows of a run
  int64_t runs;
  unsigned sum_ctas;   // CTAs that sum, all slabs together
  int64_t zero_rows;   // table rows of a zeroing CTA (0: accumulating, no zeroing)
};

// Sorted rows [run * shape.run, ...) in one group of threads; columns V per thread.
//   partial[run][0]  the piece of a token that came in from the run before
//   partial[run][1]  the piece of a token that starts in this run and goes on into the next
// U vectors per thread, a group's width apart: rows off 16-byte boundaries are read an element at a time (V = 1), and a
// thread with one column has too few bytes under way (20011 x 777 fp16 into fp32: 55 us, 62 with one; see
// launch_sum).
template <typename InT, typename OutT, int V, int U>
__global__ void __launch_bounds__(kSumThreads)
sum_rows_kernel(OutT* out, int64_t ldo, float* partial, const InT* g, int64_t ldg, const unsigned* skey,
                const unsigned* spos, int64_t n, int64_t n_cols, unsigned vocab, float scale, bool accumulate,
                SumShape shape)
{
  __shared__ unsigned char named[kSumThreads];
  grid_dep_sync();
  const int64_t nvec = n_cols / V;  // the launcher takes V = 1 unless V divides n_cols
  if (blockIdx.x >= shape.sum_ctas) {
    // rows of the table that no token names
    const int64_t v0 = int64_t(blockIdx.x - shape.sum_ctas) * shape.zero_rows;
    const int rows   = int(v0 + shape.zero_rows < int64_t(vocab) ? shape.zero_rows : int64_t(vocab) - v0);
    // first sorted position of a token >= v0: all threads probe at once, each step leaves one of 129 pieces
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t piece = (hi - lo + kSumThreads) / (kSumThreads + 1);
      const int64_t at    = lo + (int64_t(threadIdx.x) + 1) * piece - 1;
      const int below     = __syncthreads_count(at < hi && skey[at] < unsigned(v0));
      lo += int64_t(below) * piece;
      if (below < kSumThreads && lo + piece - 1 < hi) hi = lo + piece - 1;  // the next probe, which was not below
    }
    named[threadIdx.x] = 0;
    __syncthreads();
    for (int64_t i = lo + threadIdx.x; i < n; i += kSumThreads) {
      const unsigned k = skey[i];
      if (k >= unsigned(v0) + unsigned(rows)) break;
      named[k - unsigned(v0)] = 1;
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r)
      if (!named[r]) zero_row(out + (v0 + r) * ldo, n_cols, int(threadIdx.x), kSumThreads);
    return;
  }
  const int64_t gid   = (int64_t(blockIdx.x) * kSumThreads + threadIdx.x) >> shape.lg;
  const int64_t run   = gid / shape.slabs;
  const unsigned slab = unsigned(gid - run * shape.slabs);
  const int lane      = int(threadIdx.x) & ((1 << shape.lg) - 1);
  const int64_t vec   = (int64_t(slab) * U << shape.lg) + lane;  // the thread's first, the others a group's width apart
  if (run >= shape.runs || vec >= nvec) return;
  const int64_t col = vec * V;
  const int64_t lo  = run * shape.run;
  const int64_t hi  = lo + shape.run < n ? lo + shape.run : n;
  unsigned cur      = skey[lo];
  bool from_before  = lo > 0 && skey[lo - 1] == cur;
  float acc[U][V];
#pragma unroll
  for (int w = 0; w < U; ++w)
#pragma unroll
    for (int i = 0; i < V; ++i)
      acc[w][i] = 0.0f;
  const auto there = [&](int w) { return U == 1 || vec + (int64_t(w) << shape.lg) < nvec; };
  const auto away  = [&](int w) { return col + (int64_t(w) << shape.lg) * V; };
  // what has been summed of `cur`: a piece of a token that crosses an end of the run, or the whole of it
  const auto finish = [&](bool goes_on) {
#pragma unroll
    for (int w = 0; w < U; ++w) {
      if (!there(w)) continue;
      if (from_before || goes_on)
        store_partial<V>(partial + (run * 2 + (from_before ? 0 : 1)) * n_cols + away(w), acc[w]);
      else
        store_sum<OutT, V>(out + int64_t(cur) * ldo + away(w), acc[w], scale, accumulate);
    }
  };
  for (int64_t i0 = lo; i0 < hi && cur < vocab; i0 += kSumBatch) {
    // loads without conditions, so that all of them are under way at once: behind the run's end its last row again,
    // behind the last column that
    unsigned key[kSumBatch];
    Elems<InT, V> row[kSumBatch][U];
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u) {
      const int64_t i = i0 + u < hi ? i0 + u : hi - 1;
      key[u]          = skey[i];
      const InT* src  = g + int64_t(spos[i]) * ldg;
#pragma unroll
      for (int w = 0; w < U; ++w)
        row[u][w].load_once(src + (there(w) ? away(w) : col));
    }
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u) {
      if (i0 + u < hi) {
        if (key[u] != cur) {  // cur ends here
          finish(false);
          from_before = false;
          cur         = key[u];
#pragma unroll
          for (int w = 0; w < U; ++w)
#pragma unroll
            for (int i = 0; i < V; ++i)
              acc[w][i] = 0.0f;
          if (cur >= vocab) break;
        }
#pragma unroll
        for (int w = 0; w < U; ++w) {
          if (there(w)) {
            float f[V];
            row[u][w].up(f);
#pragma unroll
            for (int i = 0; i < V; ++i)
              acc[w][i] += f[i];
          }
        }
      }
    }
  }
  if (cur < vocab) finish(hi < n && skey[hi] == cur);
}

// Tokens that cross run boundaries: the group of the run in which one starts adds up its pieces in order. Few tokens do,
// and the commonest one has the most pieces, so what counts is the time of one thread's chain: four columns at most to
// a thread (shape is this kernel's own), the last run by a search of the tokens before any piece is loaded, and kFold
// pieces asked for together: 23 us of the 285 of 65536 x 4096 bf16 into 131072 rows, 37 with eight columns to a thread
// and the tokens read beside the pieces; 9.6 of the 84 of 20011 x 777 f16 into 50001 rows, 45 with sum_rows_kernel's shape.
template <typename OutT, int V>
__global__ void __launch_bounds__(kSumThreads)
fold_rows_kernel(OutT* out, int64_t ldo, const float* partial, const unsigned* skey, int64_t n, int64_t n_cols,
                 unsigned vocab, float scale, bool accumulate, SumShape shape)
{
  grid_dep_sync();
  const int64_t gid   = (int64_t(blockIdx.x) * kSumThreads + threadIdx.x) >> shape.lg;
  const int64_t run   = gid / shape.slabs;
  const unsigned slab = unsigned(gid - run * shape.slabs);
  const int lane      = int(threadIdx.x) & ((1 << shape.lg) - 1);
  const int64_t vec   = (int64_t(slab) << shape.lg) + lane;
  if (run + 1 >= shape.runs || vec >= n_cols / V) return;
  const int64_t lo   = run * shape.run;
  const int64_t hi   = lo + shape.run;  // a full run: another one follows
  const unsigned key = skey[hi - 1];
  if (key >= vocab || skey[hi] != key) return;  // nothing goes on into the next run
  if (lo > 0 && skey[lo - 1] == key) return;    // started earlier (the whole run is its)
  const int64_t col = vec * V;
  float acc[V];
  load_partial<V>(acc, partial + (run * 2 + 1) * n_cols + col);
  // The runs behind that begin with the token: the last one whose first row is the token's.
  int64_t last = run + 1;
  for (int64_t a = run + 1, b = shape.runs; b - a > 1;) {
    const int64_t mid = (a + b) >> 1;
    if (skey[mid * shape.run] <= key)
      a = last = mid;
    else
      b = mid;
  }
  const float* p     = partial + (run + 1) * 2 * n_cols + col;
  const int64_t step = 2 * n_cols;
  int64_t left       = last - run;
  for (; left >= kFold; left -= kFold, p += kFold * step) {
    float piece[kFold][V];
#pragma unroll
    for (int u = 0; u < kFold; ++u)
      load_partial<V>(piece[u], p + u * step);
#pragma unroll
    for (int u = 0; u < kFold; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i)
        acc[i] += piece[u][i];
  }
#pragma unroll 4
  for (; left > 0; --left, p += step) {
    float piece[V];
    load_partial<V>(piece, p);
#pragma unroll
    for (int i = 0; i < V; ++i)
      acc[i] += piece[i];
  }
  store_sum<OutT, V>(out + int64_t(key) * ldo + col, acc, scale, accumulate);
}

// ---------------------------------------------------------------------------------------
// Short inputs: one launch. A CTA looks after a range of the table's rows: it picks the positions that name them out of
// all tokens (read once), sorts them (by row, then by position), and its groups of threads take the rows that are named
// in turn, adding up in the order of the positions; the other rows are zeroed. No scratch. 512 tokens into 32000 x 1024
// bf16: 20.4 us, of which zeroing takes 10 at the memory's rate; every CTA picks and sorts before it writes its first
// zero. One group takes all the positions of a row: 1024 equal tokens of 4096 columns take 486 us, 1025, which are
// sorted and summed in runs, 24.
// ---------------------------------------------------------------------------------------
constexpr int kSmallThreads = 512;
constexpr int kSmallMax     = 1024;
constexpr int kSmallRows    = 128;  // of the table, per CTA at most

template <typename InT, typename OutT, typename TokT, int V>
__global__ void __launch_bounds__(kSmallThreads)
small_grad_kernel(OutT* out, int64_t ldo, const InT* g, int64_t ldg, const TokT* tokens, int n, int64_t n_cols,
                  int64_t vocab, int rows_per_cta, float scale, bool accumulate, int lg)
{
  __shared__ unsigned short found_row[kSmallMax], found_pos[kSmallMax];  // in the order of the positions
  __shared__ unsigned short pos[kSmallMax];                              // by row, then by position
  __shared__ int first[kSmallRows + 1];                                  // where a row's positions begin
  __shared__ int warp_count[kSmallThreads / 32];
  grid_dep_sync();
  constexpr int kEach = kSmallMax / kSmallThreads;  // neighbouring tokens of a thread
  const int tid = int(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int64_t v0 = int64_t(blockIdx.x) * rows_per_cta;
  const int rows   = int(v0 + rows_per_cta < vocab ? rows_per_cta : vocab - v0);
  int row[kEach], count = 0;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int i     = tid * kEach + q;
    const int64_t r = i < n ? int64_t(tokens[i]) - v0 : -1;
    row[q]          = r >= 0 && r < rows ? int(r) : -1;
    count += row[q] >= 0;
  }
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 31) warp_count[warp] = upto;
  for (int r = tid; r <= kSmallRows; r += kSmallThreads)
    first[r] = 0;
  __syncthreads();
  int at = upto - count, total = 0;
  for (int w = 0; w < kSmallThreads / 32; ++w) {
    at += w < warp ? warp_count[w] : 0;
    total += warp_count[w];
  }
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    if (row[q] >= 0) {
      found_row[at] = static_cast<unsigned short>(row[q]);
      found_pos[at] = static_cast<unsigned short>(tid * kEach + q);
      ++at;
    }
  }
  __syncthreads();
  for (int i = tid; i < total; i += kSmallThreads) {
    const int r = found_row[i];
    int before  = 0;
    for (int j = 0; j < total; ++j)
      before += found_row[j] < r || (found_row[j] == r && j < i);
    pos[before] = found_pos[i];
    atomicAdd(&first[r + 1], 1);
  }
  __syncthreads();
  if (warp == 0) {  // inclusive scan of the counts: first[r] = positions of the rows before r
    int run = 0;
    for (int b = 0; b <= rows; b += 32) {
      int c = b + lane <= rows ? first[b + lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += up;
      }
      c += run;
      if (b + lane <= rows) first[b + lane] = c;
      run = __shfl_sync(0xffffffffu, c, 31);
    }
  }
  __syncthreads();
  const int groups = kSmallThreads >> lg, group = tid >> lg, in_group = tid & ((1 << lg) - 1);
  const int64_t nvec = n_cols / V;
  for (int r = group; r < rows; r += groups) {
    const int from = first[r], to = first[r + 1];
    OutT* dst      = out + (v0 + r) * ldo;
    if (from == to) {
      if (!accumulate) zero_row(dst, n_cols, in_group, 1 << lg);
      continue;
    }
    for (int64_t vec = in_group; vec < nvec; vec += int64_t(1) << lg) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i)
        acc[i] = 0.0f;
      for (int i0 = from; i0 < to; i0 += kSumBatch) {
        Elems<InT, V> x[kSumBatch];
#pragma unroll
        for (int u = 0; u < kSumBatch; ++u)
          x[u].load_once(g + int64_t(pos[i0 + u < to ? i0 + u : to - 1]) * ldg + vec * V);
#pragma unroll
        for (int u = 0; u < kSumBatch; ++u) {
          if (i0 + u < to) {
            float f[V];
            x[u].up(f);
#pragma unroll
            for (int i = 0; i < V; ++i)
              acc[i] += f[i];
          }
        }
      }
      store_sum<OutT, V>(dst + vec * V, acc, scale, accumulate);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------
struct GradPlan {
  bool small;      // one launch, no scratch
  bool rank_sort;
  int passes, bits;
  int64_t tile;
  int tiles;
  int run;
  int64_t runs;
  size_t key_bytes;      // one array of n u32
  size_t count_bytes;    // one table of counts
  size_t partial_bytes;
  size_t total;
};

inline GradPlan plan_grad(int64_t n, int64_t n_cols, int64_t vocab)
{
  GradPlan p     = {};
  const int bits = vocab > 0 ? ilog2_floor(unsigned(vocab)) + 1 : 1;  // keys 0 .. vocab
  p.small        = n <= kSmallMax;
  p.rank_sort    = n <= kRankMax;
  p.passes       = ceil_div(bits, kRadixBits);
  p.bits         = ceil_div(bits, p.passes);
  const int sms  = sm_count();
  p.tile         = ceil_div<int64_t>(n, sms);
  if (p.tile < 2048) p.tile = 2048;
  p.tiles        = int(ceil_div<int64_t>(n > 0 ? n : 1, p.tile));
  p.run          = n >= 32768 ? 64 : (n >= 4096 ? 32 : 16);
  p.runs         = ceil_div<int64_t>(n, p.run);
  p.key_bytes    = align_up(size_t(n) * sizeof(unsigned), 256);
  p.count_bytes  = p.rank_sort ? 0 : align_up(size_t(p.tiles) << p.bits << 2, 256);
  p.partial_bytes = align_up(size_t(p.runs) * 2 * size_t(n_cols) * sizeof(float), 256);
  p.total        = p.small ? 0 : (p.rank_sort ? 2 : 4) * p.key_bytes + 2 * p.count_bytes + p.partial_bytes;
  return p;
}

inline size_t grad_scratch_bytes(int64_t n, int64_t n_cols, int64_t vocab)
{
  if (n <= 0 || n_cols <= 0 || vocab <= 0) return 0;
  return plan_grad(n, n_cols, vocab).total;
}

template <typename InT, typename OutT, int V, int U>
inline cudaError_t launch_sum(OutT* out, int64_t ldo, float* partial, const InT* g, int64_t ldg, const unsigned* skey,
                              const unsigned* spos, int64_t n, int64_t n_cols, int64_t vocab, float scale,
                              bool accumulate, const GradPlan& plan, cudaStream_t stream)
{
  SumShape s         = {};
  const int64_t nvec = n_cols / V;
  const int64_t wide = ceil_div<int64_t>(nvec, U);
  s.lg               = wide >= kSumThreads ? ilog2_floor(kSumThreads) : ilog2_floor(next_pow2(unsigned(wide)));
  const int64_t slabs = ceil_div<int64_t>(wide, int64_t(1) << s.lg);
  s.slabs            = unsigned(slabs);
  s.run              = plan.run;
  s.runs             = plan.runs;
  const int64_t sum_ctas = ceil_div<int64_t>(s.runs * slabs, kSumThreads >> s.lg);
  int64_t zero_ctas  = 0;
  if (!accumulate) {
    const int64_t row_bytes = n_cols * int64_t(sizeof(OutT));
    s.zero_rows             = (int64_t(64) << 10) / row_bytes;
    if (s.zero_rows < 1) s.zero_rows = 1;
    if (s.zero_rows > kSumThreads) s.zero_rows = kSumThreads;
    zero_ctas = ceil_div<int64_t>(vocab, s.zero_rows);
  }
  if (sum_ctas + zero_ctas > int64_t(0x7fffffff) || slabs > int64_t(0x7fffffff)) return cudaErrorInvalidValue;
  s.sum_ctas = unsigned(sum_ctas);
  if (sum_ctas + zero_ctas == 0) return cudaSuccess;
  (void)launch_dep(sum_rows_kernel<InT, OutT, V, U>, dim3(unsigned(sum_ctas + zero_ctas)), dim3(kSumThreads), 0, stream,
                   out, ldo, partial, g, ldg, skey, spos, n, n_cols, unsigned(vocab), scale, accumulate, s);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || s.runs <= 1) return e;
  constexpr int F         = V < 4 ? V : 4;
  const int64_t fold_wide = n_cols / F;
  s.lg    = fold_wide >= kSumThreads ? ilog2_floor(kSumThreads) : ilog2_floor(next_pow2(unsigned(fold_wide)));
  s.slabs = unsigned(ceil_div<int64_t>(fold_wide, int64_t(1) << s.lg));
  const int64_t fold_ctas = ceil_div<int64_t>(s.runs * s.slabs, kSumThreads >> s.lg);
  if (fold_ctas > int64_t(0x7fffffff)) return cudaErrorInvalidValue;
  (void)launch_dep(fold_rows_kernel<OutT, F>, dim3(unsigned(fold_ctas)), dim3(kSumThreads), 0, stream, out, ldo,
                   partial, skey, n, n_cols, unsigned(vocab), scale, accumulate, s);
  return cudaGetLastError();
}

template <typename InT, typename OutT, typename TokT, int V>
inline cudaError_t launch_small(OutT* out, int64_t ldo, const InT* g, int64_t ldg, const TokT* tokens, int n,
                                int64_t n_cols, int64_t vocab, float scale, bool accumulate, cudaStream_t stream)
{
  const int64_t nvec = n_cols / V;
  const int lg       = nvec >= 128 ? 7 : ilog2_floor(next_pow2(unsigned(nvec)));
  // ranges of some 64 KB of the table, but at least two CTAs per SM
  int64_t rows       = (int64_t(64) << 10) / (n_cols * int64_t(sizeof(OutT)));
  const int64_t most = ceil_div<int64_t>(vocab, 2 * int64_t(sm_count()));
  rows               = rows < most ? rows : most;
  rows               = rows < 1 ? 1 : (rows > kSmallRows ? kSmallRows : rows);
  const int64_t ctas = ceil_div<int64_t>(vocab, rows);
  (void)launch_dep(small_grad_kernel<InT, OutT, TokT, V>, dim3(unsigned(ctas)), dim3(kSmallThreads), 0, stream, out, ldo,
                   g, ldg, tokens, n, n_cols, vocab, int(rows), scale, accumulate, lg);
  return cudaGetLastError();
}

template <typename InT, typename OutT, typename TokT>
inline cudaError_t launch_grad(OutT* out, int64_t ldo, const InT* g, int64_t ldg, const TokT* tokens, int64_t n,
                               int64_t n_cols, int64_t vocab, float scale, bool accumulate, cudaStream_t stream,
                               Workspace ws)
{
  if (n_cols <= 0 || vocab <= 0) return cudaSuccess;
  if (n <= 0 && accumulate) return cudaSuccess;
  constexpr int V = 16 / int(sizeof(InT));  // 16-byte loads; outputs of V elements
  const int need  = common_alignment({reinterpret_cast<uintptr_t>(g), uintptr_t(ldg) * sizeof(InT)});
  const int want  = V * int(sizeof(OutT));
  const int have  = common_alignment({reinterpret_cast<uintptr_t>(out), uintptr_t(ldo) * sizeof(OutT)});
  const bool vectors = need >= 16 && have >= want && n_cols % V == 0;
  const GradPlan plan = plan_grad(n, n_cols, vocab);
  if (plan.small)
    return vectors ? launch_small<InT, OutT, TokT, V>(out, ldo, g, ldg, tokens, int(n), n_cols, vocab, scale, accumulate, stream)
                   : launch_small<InT, OutT, TokT, 1>(out, ldo, g, ldg, tokens, int(n), n_cols, vocab, scale, accumulate, stream);
  Scratch scratch(ws, plan.total, stream);
  if (scratch.error() != cudaSuccess) return scratch.error();
  char* at        = static_cast<char*>(scratch.get());
  unsigned* key0  = reinterpret_cast<unsigned*>(at);
  unsigned* pos0  = reinterpret_cast<unsigned*>(at + plan.key_bytes);
  at += 2 * plan.key_bytes;
  cudaError_t e = cudaSuccess;
  if (n > 0 && plan.rank_sort) {
    const int padded  = int(ceil_div<int64_t>(n, 4 * kRankLanes)) * 4 * kRankLanes;
    const unsigned gr = unsigned(ceil_div<int64_t>(n, kRankThreads / kRankLanes));
    (void)launch_dep(rank_sort_kernel<TokT>, dim3(gr), dim3(kRankThreads), size_t(padded) * 4, stream, key0, pos0,
                     tokens, int(n), unsigned(vocab));
    e = cudaGetLastError();
  } else if (n > 0) {
    unsigned* key1 = reinterpret_cast<unsigned*>(at);
    unsigned* pos1 = reinterpret_cast<unsigned*>(at + plan.key_bytes);
    at += 2 * plan.key_bytes;
    unsigned* count[2] = {reinterpret_cast<unsigned*>(at), reinterpret_cast<unsigned*>(at + plan.count_bytes)};
    at += 2 * plan.count_bytes;
    const dim3 grid(unsigned(plan.tiles)), block(kRadixThreads);
    (void)launch_dep(radix_count_kernel<TokT>, grid, block, 0, stream, count[0], count[1], tokens, n, plan.tile,
                     unsigned(vocab), plan.bits);
    e                  = cudaGetLastError();
    unsigned *k[2]     = {key0, key1}, *p[2] = {pos0, pos1};
    int from           = 1;
    for (int pass = 0; pass < plan.passes && e == cudaSuccess; ++pass) {
      const bool more  = pass + 1 < plan.passes;
      const int to     = 1 - from;
      unsigned* counts = count[pass & 1];
      unsigned* next   = more ? count[1 - (pass & 1)] : nullptr;
      if (pass >= 1 && more) {  // the table that the first pass cleared has been used: clear the other one
        e = cudaMemsetAsync(next, 0, plan.count_bytes, stream);
        if (e != cudaSuccess) break;
      }
      (void)launch_dep(radix_scatter_kernel<TokT>, grid, block, 0, stream, k[to], p[to],
                       pass == 0 ? tokens : nullptr, k[from], p[from], counts, next, n, plan.tile, unsigned(vocab),
                       pass * plan.bits, plan.bits);
      e    = cudaGetLastError();
      from = to;
    }
    key0 = k[from];
    pos0 = p[from];
  }
  if (e != cudaSuccess) return e;
  float* partial  = reinterpret_cast<float*>(at);
  if (vectors)
    return launch_sum<InT, OutT, V, 1>(out, ldo, partial, g, ldg, key0, pos0, n, n_cols, vocab, scale, accumulate, plan,
                                       stream);
  return launch_sum<InT, OutT, 1, 4>(out, ldo, partial, g, ldg, key0, pos0, n, n_cols, vocab, scale, accumulate, plan,
                                     stream);
}

}  // namespace emb
}  // namespace detail
}  // namespace raft_b200
