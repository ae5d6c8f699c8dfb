// One token per row of logits by temperature, top-k, top-p and min-p, from a given uniform number.
//
// With z the row's logits, zmax the largest, T the temperature and w_v = exp((z_v - zmax) / T), tokens are ordered by
// falling logit, equal logits by rising token. Kept are the first top_k of that order, of those the tokens with
// w >= min_p, and of those the shortest beginning of the order whose weight reaches top_p of their whole weight. Drawn
// is the first kept token, BY TOKEN, at which the running weight exceeds u times the kept weight. T <= 0 takes the
// largest logit (the lowest token of equals). NaN logits count as -inf; a row of nothing else has no token: -1.
//
// Which side of a border a token falls on is decided by sums over the vocabulary in which a token may weigh 1e-6 of
// the whole, so weights are computed in fp64 and summed as INTEGERS of 2^-shift, shift = 62 - ceil(log2 vocab) but at
// most kMaxShift (45 bits for 131072 tokens): exact, the same whatever the order, the split of the row or the number of
// rows of the call.
//
// A cluster of CTAs takes a row, every CTA a part, which it keeps in shared memory. What is kept is nearly always a short
// beginning of the order, and the work is in not touching the rest more than once or twice, two elements at a time:
//   - every thread takes the maximum of its elements. The maxima are counted over the cluster by their keys (the logits'
//     bits, made to rise with their value), in bins of 1/128 octave from the largest down: where n maxima lie at or
//     above a bound there are at least n such elements, so the bin of the top_k-th maximum bounds the first top_k
//     elements from below, and min_p is a bound by itself. For a top-p alone, beginnings that hold kShort / 2 and
//     kList / 2 maxima are tried: whether their weight is enough is seen when the row's whole weight is summed, which a
//     top-p needs anyway.
//   - the elements above the bound, if they are at most kList, are collected in the first CTA, sorted, and the rest
//     happens there; the other CTAs are done.
// Longer beginnings (a flat distribution, a large k) are narrowed by radix selection over all elements, a digit at a
// time, by counts or weights summed over the cluster through distributed shared memory, and drawn from in place: 256 rows
// of 131072 bf16 with a top-k of 50 take 54 us, with a top-p of 0.9 over a body of thousands of tokens 452 (fp32: 98, 608).
// The bins are of keys, not of values, and end 16 octaves below the largest logit, at zero at the latest: where a row's
// largest logit is 0 (its maximum subtracted) or little above, few maxima lie in them, no bound is found, and the row
// takes the long way, or the slow sort below: results are the same, the top-k of 50 takes 199 us (fp32: 340).
#pragma once

#include "launch.cuh"
#include "topk_distill.cuh"  // RowPart, cluster primitives

#include <cfloat>

namespace raft_b200 {
namespace detail {
namespace sample {

using distill::RowPart;
using u64 = unsigned long long;

constexpr int kThreads    = 512;
constexpr int kWarps      = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kDigitBits  = 11;
constexpr int kBins       = 1 << kDigitBits;
constexpr int kMaxPartKb  = 160;  // of a row in a CTA's shared memory
constexpr int kList       = 2048;
constexpr int kShort      = 256;  // up to here a list is sorted by comparing all pairs
constexpr int kScratch    = kList * 12;  // bytes of the row's place in shared memory at least: the sort of a list
constexpr int kMaxVocab   = 1 << 24;  // the sums of 32 vectors of the largest part (131 KB) fit beside the rest
constexpr int kMaxShift   = 50;  // weights below 2^51, so that an addition rounds them to integers

template <typename T>
struct Args {
  const T* logits;
  int64_t ldl;
  const float* uniform;
  const float* temperature;  // each may be null: the value for all rows counts then
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  void* out;
  int out64;
  float* logprobs;  // may be null
  int64_t n_rows;
  int vocab;
  int per_cta;  // vectors of a row per CTA
  int shift;    // weights are integers of 2^-shift
  int row_bytes;  // of the row's place in shared memory
};

// An element as an unsigned number of its own width that rises with its value: half the range plus or minus the bits
// of its magnitude, so that -0 and +0 are one; NaN as -inf. Keys are packed as the elements were.
template <typename T, int kBits_, unsigned kInf>
struct KeyOf {
  static constexpr int kBits        = kBits_;
  static constexpr unsigned kZero   = 1u << (kBits - 1);
  static constexpr unsigned kNegInf = kZero - kInf;

  B2R_DI static unsigned of_bits(unsigned b)  // bits of an element
  {
    const unsigned mag = b & (kZero - 1u);
    const unsigned key = (b & kZero) ? kZero - mag : kZero + mag;
    return mag > kInf ? kNegInf : key;
  }
  B2R_DI static Words4 pack(const Words4& v)
  {
    Words4 r;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      r.w[q] = kBits == 32 ? of_bits(v.w[q]) : (of_bits(v.w[q] & 0xffffu) | (of_bits(v.w[q] >> 16) << 16));
    return r;
  }
  B2R_DI static unsigned at(const Words4& v, int e)
  {
    if constexpr (kBits == 32)
      return v.w[e];
    else
      return (e & 1) ? v.w[e / 2] >> 16 : v.w[e / 2] & 0xffffu;
  }
  B2R_DI static float value(unsigned k)
  {
    const int d         = int(k - kZero);
    const unsigned bits = d < 0 ? (unsigned(-d) | kZero) : unsigned(d);
    if constexpr (kBits == 32) {
      return __uint_as_float(bits);
    } else {
      const uint16_t b = uint16_t(bits);
      T x;
      memcpy(&x, &b, 2);
      return FloatIo<T>::up(x);
    }
  }
  // bits of element e
  B2R_DI static unsigned bits_at(const Words4& v, int e) { return at(v, e); }
  // element e as fp32 (NaN as it is)
  B2R_DI static float float_at(const Words4& v, int e)
  {
    const float2 f = up_pair<T>(v, e / 2);
    return (e & 1) ? f.y : f.x;
  }
  // the larger ones of two words' elements (NaN loses)
  B2R_DI static uint32_t larger(uint32_t a, uint32_t b)
  {
    if constexpr (kBits == 32) {
      return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
      using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      Pair x, y;
      memcpy(&x, &a, 4);
      memcpy(&y, &b, 4);
      x = __hmax2(x, y);
      memcpy(&a, &x, 4);
      return a;
    }
  }
  B2R_DI static Words4 larger(const Words4& a, const Words4& b)
  {
    Words4 r;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      r.w[q] = larger(a.w[q], b.w[q]);
    return r;
  }
  // the largest element as fp32 (NaN only if all are)
  B2R_DI static float largest(const Words4& v)
  {
    Words<1> m;
    m.w[0] = larger(larger(v.w[0], v.w[1]), larger(v.w[2], v.w[3]));
    if constexpr (kBits == 32) {
      return __uint_as_float(m.w[0]);
    } else {
      const float2 f = up_pair<T>(m, 0);
      return fmaxf(f.x, f.y);
    }
  }
  // key of a value that an element of T can have
  B2R_DI static unsigned of_value(float x)
  {
    if constexpr (kBits == 32) {
      return of_bits(__float_as_uint(x));
    } else {
      const T h = FloatIo<T>::down(x);
      uint16_t b;
      memcpy(&b, &h, 2);
      return of_bits(b);
    }
  }
  // lowest key whose value is at least x
  B2R_DI static unsigned at_least(double x)
  {
    if constexpr (kBits == 32) {
      return of_bits(__float_as_uint(__double2float_ru(x)));
    } else {  // by bisection of the keys, whose values rise
      unsigned lo = kNegInf, hi = kZero + kInf;  // -inf ... +inf
      while (lo < hi) {
        const unsigned mid = (lo + hi) >> 1;
        if (double(value(mid)) >= x)
          hi = mid;
        else
          lo = mid + 1;
      }
      return lo;
    }
  }
};
template <typename T>
struct Key;
template <>
struct Key<float> : KeyOf<float, 32, 0x7f800000u> {};
template <>
struct Key<__half> : KeyOf<__half, 16, 0x7c00u> {};
template <>
struct Key<__nv_bfloat16> : KeyOf<__nv_bfloat16, 16, 0x7f80u> {};

// 2^(i / 32)
__constant__ const double kPowers[32] = {
  1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
  1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
  1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
  1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
  1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
  1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
  1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
  1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};

B2R_DI u64 warp_sum_u64(u64 v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v += __shfl_xor_sync(distill::kFull, v, o);
  return v;
}
B2R_DI u64 warp_scan_u64(u64 v)  // inclusive
{
  const int lane = int(threadIdx.x) & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(distill::kFull, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
B2R_DI void cluster_store_u64(u64* p, unsigned rank, u64 v)
{
  const unsigned local = smem_u32(p);
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(v) : "memory");
}
B2R_DI unsigned cluster_load_u32(const unsigned* p, unsigned rank)
{
  const unsigned local = smem_u32(p);
  unsigned remote, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}
B2R_DI unsigned cluster_address(const void* p, unsigned rank)
{
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  return remote;
}
B2R_DI void cluster_add_u32(unsigned* p, unsigned rank, unsigned v)
{
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(cluster_address(p, rank)), "r"(v) : "memory");
}
B2R_DI void cluster_max_u32(unsigned* p, unsigned rank, unsigned v)
{
  asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(cluster_address(p, rank)), "r"(v) : "memory");
}
B2R_DI void cluster_sync()
{
  distill::cluster_arrive();
  distill::cluster_wait();
}

B2R_HDI constexpr int bins_of(int size) { return kBins / size > kList ? kBins / size : kList; }

template <typename T, bool kCached>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  using K          = Key<T>;
  extern __shared__ __align__(16) unsigned char sample_smem[];
  __shared__ __align__(16) unsigned hist[2][kBins];  // counts of this CTA and of the row; words of the bins' sums
  __shared__ double powers[32];                 // 2^(i / 32)
  __shared__ unsigned kmax_all, list_at;
  __shared__ u64 posted[4][4][kMaxCluster];     // up to four values of every CTA, four exchanges deep
  __shared__ u64 result[2][2];
  __shared__ u64 warp_part[4][kWarps];
  __shared__ u64 carry;
  Words4* slice = reinterpret_cast<Words4*>(sample_smem);  // [per_cta] if kCached
  const unsigned rank = distill::cluster_rank();
  const unsigned size = distill::cluster_size();
  // sums over the cluster of the bins this CTA looks after; the list
  u64* bins        = reinterpret_cast<u64*>(sample_smem + a.row_bytes);  // [bins_of(size)]
  u64* units       = bins + bins_of(int(size));                                  // sums of 32 vectors each, in order
  unsigned* totals = hist[1];
  const int tid = int(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  grid_dep_sync();
  const int64_t row = int64_t(blockIdx.x) / size;
  const T* z        = a.logits + row * a.ldl;
  const RowPart<T> part(z, a.vocab, int(rank) * a.per_cta, a.per_cta);
  if constexpr (kCached) {  // every thread its own vectors, all of them under way at once
    for (int j = tid; j < part.n; j += kThreads) {
      if (part.whole(j))
        distill::copy_async16(slice + j, part.at + j * VE);
      else
        slice[j] = part.load_edge(j);
    }
    distill::copy_commit();
  }
  for (int i = tid; i < kBins / 4; i += kThreads)
    reinterpret_cast<uint4*>(hist[0])[i] = reinterpret_cast<uint4*>(totals)[i] = make_uint4(0, 0, 0, 0);
  if (tid < 32) powers[tid] = kPowers[tid];
  if (tid == 0) kmax_all = list_at = 0;
  __syncthreads();
  distill::cluster_arrive();  // every CTA of the cluster has started and is set up
  const float temp   = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  const int top_k    = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  const float top_p  = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  const float min_p  = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  const float u      = a.uniform[row];
  const bool greedy  = !(temp > 0.0f);
  const auto raw     = [&](int j) { return kCached ? slice[j] : part.load(j); };
  const auto vec     = [&](int j) { return K::pack(raw(j)); };  // keys
  int exchanges      = 0;

  auto write = [&](int64_t token, float logprob) {  // by one thread of the cluster
    if (a.out64)
      static_cast<long long*>(a.out)[row] = token;
    else
      static_cast<int*>(a.out)[row] = int(token);
    if (a.logprobs != nullptr) a.logprobs[row] = logprob;
  };
  // every CTA's values, known to all afterwards (four calls long)
  auto post4 = [&](const u64 (&v)[4]) {
    auto slot = posted[exchanges & 3];
    ++exchanges;
    if (tid < int(size)) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        cluster_store_u64(&slot[q][rank], unsigned(tid), v[q]);
    }
    cluster_sync();
    return slot;
  };
  auto post = [&](u64 v) {
    u64* slot = posted[exchanges & 3][0];
    ++exchanges;
    if (tid < int(size)) cluster_store_u64(&slot[rank], unsigned(tid), v);
    cluster_sync();
    return slot;
  };
  auto block_sum = [&](u64 v) {  // to all threads
    v = warp_sum_u64(v);
    __syncthreads();
    if (lane == 0) warp_part[0][warp] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      s += warp_part[0][w];
    return s;
  };

  // the row; every thread's largest element, and the row's
  const bool by_k   = !greedy && top_k > 0 && top_k < a.vocab;
  const bool by_p   = !greedy && top_p < 1.0f;
  const bool by_min = !greedy && min_p > 0.0f;
  Words4 mine_max    = distill::minus_inf<T>();
  if constexpr (kCached) distill::copy_wait<0>();
  for (int j = tid; j < part.n; j += kThreads)
    mine_max = K::larger(mine_max, raw(j));
  unsigned kmax = K::of_value(K::largest(mine_max));
  const unsigned own_max = kmax;
  kmax = __reduce_max_sync(distill::kFull, kmax);
  distill::cluster_wait();
  if (lane < int(size)) cluster_max_u32(&kmax_all, unsigned(lane), kmax);
  cluster_sync();
  kmax = kmax_all;
  if (kmax <= K::kNegInf) {  // nothing to draw from
    if (rank == 0 && tid == 0) write(-1, -INFINITY);
    return;
  }
  // f(vector, its first token) for the vectors that hold an element of at least `bound`
  const auto vectors_from = [&](float bound, auto f) {
    for (int j = tid; j < part.n; j += kThreads) {
      const Words4 v = raw(j);
      if (K::largest(v) >= bound) f(v, part.first + j * VE);
    }
  };
  if (greedy) {  // the lowest token of those with the largest key
    const float top = K::value(kmax);
    unsigned token0 = 0xffffffffu;
    vectors_from(top, [&](const Words4& v, int token) {
#pragma unroll
      for (int e = VE - 1; e >= 0; --e)
        if (K::float_at(v, e) == top) token0 = min(token0, unsigned(token + e));
    });
    token0 = __reduce_min_sync(distill::kFull, token0);
    if (lane == 0) warp_part[0][warp] = token0;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w)
      token0 = min(token0, unsigned(warp_part[0][w]));
    const u64* all = post(token0);
    for (unsigned r = 0; r < size; ++r)
      token0 = min(token0, unsigned(all[r]));
    if (rank == 0 && tid == 0) write(int64_t(token0), 0.0f);
    return;
  }
  // 2^x by table and polynomial: x * 32 = n + r, 2^x = 2^(n / 32) 2^(r / 32), the second by its Taylor series to the
  // fifth power, the first from `powers` and an exponent (P. T. P. Tang, 1989). With |r / 32 ln 2| <= ln 2 / 64 the
  // series is off by 2.3e-15 of its value, the roundings by four of 2^-53 and, for the exponent's (difference, slope and
  // product), |ln w| 2^-51: no weight by more than 2^-48 of the largest, before it is rounded to an integer. What
  // rounds to 0 is cut off at `low` (and NaN there is none); temperatures above 1e30 count as that.
  const double zmax    = double(K::value(kmax));
  const double slope   = 1.4426950408889634 / double(fminf(temp, 1e30f));
  const double slope32 = slope * 32.0;
  const int shift      = a.shift;
  const float top      = K::value(kmax);
  const float cut      = __double2float_rd(zmax - double(shift + 2) / slope);
  // no other logit counts: a +inf one, or floats further apart than the cut
  const bool sharp     = top == INFINITY || cut >= nextafterf(top, -INFINITY);
  const bool bottom    = cut < -FLT_MAX;  // logits near the lowest value: -inf has to be told from what counts
  const float low      = fmaxf(cut, -FLT_MAX);
  const bool special   = sharp || bottom;
  const auto weight_of = [&](float z) -> u64 {
    const double y   = (double(fmaxf(z, low)) - zmax) * slope32;
    const double big = y + 6755399441055744.0;  // 1.5 * 2^52: the nearest integer in the low bits
    const int n      = __double2loint(big);
    const double r   = (y - (big - 6755399441055744.0)) * (0.6931471805599453 / 32.0);
    double p         = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p                = fma(p, r, 1.0 / 6.0);
    p                = fma(p, r, 0.5);
    p                = fma(p, r, 1.0);
    p                = fma(p, r, 1.0);
    const double w   = p * powers[n & 31];
    const double s   = __hiloint2double(__double2hiint(w) + (((n >> 5) + shift) << 20), __double2loint(w));
    const u64 whole  = u64(__double_as_longlong(s + 4503599627370496.0)) & 0xfffffffffffffull;  // 2^52: to an integer
    if (!special) return whole;
    return sharp ? (z == top ? u64(1) << shift : 0) : (z >= -FLT_MAX ? whole : 0);
  };
  const auto weight = [&](unsigned key) { return weight_of(K::value(key)); };

  // kept: key > tau, or key == tau and token <= last
  unsigned tau = K::kNegInf + 1;
  int last     = 0x7fffffff;
  const auto kept = [&](unsigned key, int token) { return key > tau || (key == tau && token <= last); };

  // Sums of value(vector, element, token) over runs of 32 vectors; *before: of the CTAs ahead of this one. Returns the whole sum.
  auto sum_in_order = [&](auto value, u64* before, u64* mine) {
    u64 own = 0;
    for (int j0 = warp * 32; j0 < part.n; j0 += kThreads) {
      u64 s = 0;
      if (j0 + lane < part.n) {
        const Words4 v = raw(j0 + lane);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          s += value(v, e, part.first + (j0 + lane) * VE + e);
      }
      s = warp_sum_u64(s);
      if (lane == 0) units[j0 / 32] = s;
      own += s;
    }
    __syncthreads();
    if (lane == 0) warp_part[0][warp] = own;
    __syncthreads();
    own = 0;
    for (int w = 0; w < kWarps; ++w)
      own += warp_part[0][w];
    const u64* all = post(own);
    u64 total = 0, ahead = 0;
    for (unsigned r = 0; r < size; ++r) {
      total += all[r];
      ahead += r < rank ? all[r] : 0;
    }
    *before = ahead;
    *mine   = own;
    return total;
  };
  // by warp 0 of the CTA whose range holds `target` (relative to the CTA's own beginning): the token at which the
  // running sum exceeds it, and that token's key
  auto locate = [&](auto value, u64 target, unsigned* key) {
    const int n_units = (part.n + 31) / 32;
    u64 run = 0;
    int at  = 0;
    for (int b = 0; b < n_units; b += 32) {
      const u64 s    = b + lane < n_units ? units[b + lane] : 0;
      const u64 incl = run + warp_scan_u64(s);
      const unsigned over = __ballot_sync(distill::kFull, incl > target);
      if (over != 0u) {
        const int l = __ffs(int(over)) - 1;
        at          = b + l;
        run         = __shfl_sync(distill::kFull, incl - s, l);
        break;
      }
      run = __shfl_sync(distill::kFull, incl, 31);
    }
    const int j = at * 32 + lane;
    Words4 v    = distill::minus_inf<T>();
    u64 s       = 0;
    if (j < part.n) {
      v = raw(j);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        s += value(v, e, part.first + j * VE + e);
    }
    const u64 incl      = run + warp_scan_u64(s);
    const unsigned over = __ballot_sync(distill::kFull, incl > target);
    const int l         = __ffs(int(over)) - 1;
    u64 upto            = incl - s;
    int token           = -1;
    unsigned found      = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int t = part.first + j * VE + e;
      upto += value(v, e, t);
      if (token < 0 && upto > target) {
        token = t;
        found = K::of_bits(K::bits_at(v, e));
      }
    }
    *key = __shfl_sync(distill::kFull, found, l);
    return __shfl_sync(distill::kFull, token, l);
  };
  // The border of the order at which the sum of value(key) over the kept tokens reaches `target` (at least 1, at most
  // the whole sum): its key in *border, the sum over larger keys in *above. With kCount the values are 1.
  // A target above the whole sum, which is returned in *total: the border is below every kept key, false.
  auto select = [&](auto count, auto value, auto target_of, unsigned* border, u64* above, u64* total) {
    constexpr bool kCount = decltype(count)::value;
    unsigned prefix = 0;  // bits of the border found so far
    int left        = K::kBits;
    u64 over        = 0;
    u64 target      = 0;
    while (left > 0) {
      const int bits  = left > kDigitBits ? kDigitBits : left;
      const int shift = left - bits;
      const int n     = 1 << bits;
      for (int i = tid; i < n; i += kThreads)
        hist[0][i] = hist[1][i] = 0;
      __syncthreads();
      for (int j = tid; j < part.n; j += kThreads) {
        const Words4 v = vec(j);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const unsigned key = K::at(v, e);
          if ((left == K::kBits || (key >> left) == prefix) && kept(key, part.first + j * VE + e)) {
            const unsigned d = (key >> shift) & unsigned(n - 1);
            if constexpr (kCount) {
              atomicAdd(&hist[0][d], 1u);
            } else {
              const u64 w = value(key);
              if (w != 0) {  // a 64-bit sum by its words: the low one tells when it wraps
                const unsigned lo   = unsigned(w);
                const unsigned old  = atomicAdd(&hist[0][d], lo);
                const unsigned high = unsigned(w >> 32) + (old + lo < old ? 1u : 0u);
                if (high != 0u) atomicAdd(&hist[1][d], high);
              }
            }
          }
        }
      }
      // this CTA's share of the bins, over the cluster; bins fall with the rank, as the order does
      cluster_sync();
      const int own_bins = n / int(size);
      const int top      = n - 1 - int(rank) * own_bins;  // its largest
      u64 mine           = 0;
      for (int i = tid; i < own_bins; i += kThreads) {
        u64 s = 0;
        for (unsigned r = 0; r < size; ++r) {
          s += cluster_load_u32(&hist[0][top - i], r);
          if (!kCount) s += u64(cluster_load_u32(&hist[1][top - i], r)) << 32;
        }
        bins[i] = s;
        mine += s;
      }
      mine           = block_sum(mine);
      const u64* all = post(mine);
      u64 whole = 0, ahead = over;
      for (unsigned r = 0; r < size; ++r) {
        whole += all[r];
        ahead += r < rank ? all[r] : 0;
      }
      if (left == K::kBits) {
        *total = whole;
        target = target_of(whole);
        if (target > whole) return false;
      }
      u64* res = result[(K::kBits - left) / kDigitBits & 1];
      if (ahead < target && target <= ahead + mine && warp == 0) {  // the border is in one of this CTA's bins
        u64 run = ahead;
        for (int b = 0; b < own_bins; b += 32) {
          const u64 s         = b + lane < own_bins ? bins[b + lane] : 0;
          const u64 incl      = run + warp_scan_u64(s);
          const unsigned full = __ballot_sync(distill::kFull, incl >= target);
          if (full != 0u) {
            const int l       = __ffs(int(full)) - 1;
            const u64 before  = __shfl_sync(distill::kFull, incl - s, l);
            const unsigned bin = unsigned(top - b - l);
            if (lane < int(size)) {
              cluster_store_u64(&res[0], unsigned(lane), bin);
              cluster_store_u64(&res[1], unsigned(lane), before);
            }
            break;
          }
          run = __shfl_sync(distill::kFull, incl, 31);
        }
      }
      cluster_sync();
      prefix = (prefix << bits) | unsigned(res[0]);
      over   = res[1];
      left   = shift;
    }
    *border = prefix;
    *above  = over;
    return true;
  };
  // the token of the `nth` (from 1) kept element whose key is tau, as a limit for all CTAs
  auto limit_ties = [&](u64 nth) {
    const auto is_tie = [&](const Words4& v, int e, int token) -> u64 {
      return K::of_bits(K::bits_at(v, e)) == tau && token <= last ? 1 : 0;
    };
    u64 before, mine;
    const u64 total = sum_in_order(is_tie, &before, &mine);
    if (nth >= total) return;  // all of them
    u64 found = 0;
    if (before < nth && nth <= before + mine) {
      if (warp == 0) {
        unsigned key;
        found = u64(locate(is_tie, nth - 1 - before, &key)) + 1;
        if (lane == 0) carry = found;
      }
      __syncthreads();
      found = carry;
    }
    const u64* all = post(found);
    for (unsigned r = 0; r < size; ++r)
      if (all[r] != 0) last = int(all[r]) - 1;
  };

  // w >= min_p, as a bound on the key
  const double mp     = min_p < 1.0f ? double(min_p) : 1.0;
  const unsigned kmin = !by_min ? 0u : (mp == 1.0 ? kmax : min(kmax, K::at_least(zmax + log2(mp) / slope)));
  // elements of at least `bound` in this CTA
  const auto count_from = [&](float bound) {
    u64 n = 0;
    vectors_from(bound, [&](const Words4& v, int) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        n += K::float_at(v, e) >= bound ? 1 : 0;
    });
    return block_sum(n);
  };
  // Threads' maxima by their distance from the largest key, in bins of 2^kFine keys (a 128th of an octave; the last bin
  // holds all that lie further down).
  constexpr int kFine = K::kBits == 32 ? 16 : (std::is_same<T, __half>::value ? 3 : 0);
  if (by_k || (by_p && !by_min)) {
    if (own_max > K::kNegInf) atomicAdd(&hist[0][min((kmax - own_max) >> kFine, unsigned(kBins - 1))], 1u);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) {
      const unsigned n = hist[0][i];
      if (n != 0)
        for (unsigned r = 0; r < size; ++r)
          cluster_add_u32(&totals[i], r, n);
    }
    cluster_sync();
  }
  const float lowest = K::value(K::kNegInf + 1);
  // A bound at or above which there are at least `goal` threads' maxima (the lowest value: there are fewer in all).
  const auto bound_of = [&](u64 goal) {
    constexpr int kEach = kBins / kThreads;
    u64 s               = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q)
      s += totals[tid * kEach + q];
    const u64 incl = warp_scan_u64(s);
    __syncthreads();
    if (lane == 31) warp_part[0][warp] = incl;
    if (tid == 0) carry = kBins - 1;
    __syncthreads();
    u64 run = incl - s;
    for (int w = 0; w < warp; ++w)
      run += warp_part[0][w];
    if (run < goal && goal <= run + s) {
      int q = 0;
      while ((run += totals[tid * kEach + q]) < goal)
        ++q;
      carry = u64(tid * kEach + q);
    }
    __syncthreads();
    const unsigned down = (unsigned(carry) + 1) << kFine;  // the bin's lowest key is kmax - down + 1
    const bool last_bin = carry == kBins - 1;
    return last_bin || kmax < K::kNegInf + down ? lowest : K::value(kmax - down + 1);
  };
  // Draws from the n elements of at least `bound`, collected in the first CTA; `base` of them are in the CTAs ahead.
  // `whole`: the weight of all tokens that top-p is measured by, or 0: that of those top_k and min-p leave.
  auto draw_from_list = [&](float bound, int n, int base, u64 whole) {
    vectors_from(bound, [&](const Words4& v, int first) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (K::float_at(v, e) >= bound) {
          // larger keys first, lower tokens first among equals
          cluster_store_u64(&bins[base + int(atomicAdd(&list_at, 1u))], 0,
                            (u64(K::of_bits(K::bits_at(v, e))) << 32) | (0xffffffffu - unsigned(first + e)));
        }
      }
    });
    cluster_sync();
    if (rank != 0) return;
    u64* list    = bins;
    u64* weights = reinterpret_cast<u64*>(&hist[0][0]);  // [kList]
    // Falling order of list[0 .. count), no two of which are equal. bin_of(x), below kList, never falls as x does.
    const auto sort = [&](int count, auto bin_of) {
      constexpr int kEach = kList / kThreads;
      if (count <= kShort) {  // the place of a token is the number of larger ones
        __syncthreads();
        const u64 mine = tid < count ? list[tid] : 0;
        if (tid == count && (count & 1)) list[tid] = 0;
        __syncthreads();
        int place = 0;
        for (int i = 0; i < count; i += 2) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list + i);
          place += (x.x > mine ? 1 : 0) + (x.y > mine ? 1 : 0);
        }
        __syncthreads();
        if (tid < count) list[place] = mine;
        __syncthreads();
        return;
      }
      // into bins, by counts; then every token looks for its place among those of its bin, nearly always a few (a
      // sorting network over 2048 places takes 14 us, mostly shuffles; this 2). Where no bound was found the bins span
      // the type's whole range and one holds all, so that all pairs are compared: 256 x 2000 fp32, top-k 1000, 223 us.
      u64* spread     = reinterpret_cast<u64*>(sample_smem);              // [kList]
      unsigned* start = reinterpret_cast<unsigned*>(spread + kList);      // [kList]
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        start[tid + q * kThreads] = 0;
      __syncthreads();
      u64 x[kEach];
      unsigned bin[kEach], at[kEach];
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        const int i = tid + q * kThreads;
        if (i < count) {
          x[q]   = list[i];
          bin[q] = bin_of(x[q]);
          at[q]  = atomicAdd(&start[bin[q]], 1u);
        }
      }
      __syncthreads();
      unsigned n_bin[kEach], sum = 0;
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        n_bin[q] = sum;
        sum += start[tid * kEach + q];
      }
      const u64 incl = warp_scan_u64(sum);
      if (lane == 31) warp_part[0][warp] = incl;
      __syncthreads();
      u64 base = incl - sum;
      for (int w = 0; w < warp; ++w)
        base += warp_part[0][w];
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        start[tid * kEach + q] = unsigned(base) + n_bin[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        if (tid + q * kThreads < count) spread[start[bin[q]] + at[q]] = x[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        if (tid + q * kThreads < count) {
          const unsigned from = start[bin[q]];
          const unsigned to   = bin[q] + 1 < unsigned(kList) ? start[bin[q] + 1] : unsigned(count);
          unsigned place      = from;
          for (unsigned i = from; i < to; ++i)
            place += spread[i] > x[q] ? 1u : 0u;
          list[place] = x[q];
        }
      }
      __syncthreads();
    };
    // by value: even steps from the largest logit down to the bound
    const float step_v = top > bound ? float(kList - 1) / (top - bound) : 0.0f;
    const auto value_bin = [&](u64 x) {
      const float z = K::value(unsigned(x >> 32));
      const float d = z == top ? 0.0f : (top - z) * step_v;  // (0 * inf is NaN: the first bin)
      return d > 0.0f ? min(unsigned(d), unsigned(kList - 1)) : 0u;
    };
    const auto token_bin = [&](u64 x) {
      return unsigned(u64(0xffffffffu - unsigned(x >> 32)) * unsigned(kList) / unsigned(a.vocab));
    };
    sort(n, value_bin);
    int m = by_k && top_k < n ? top_k : n;
    // running weights of the first m that min-p leaves (from it on all are below): four places per thread
    constexpr int kEach = kList / kThreads;
    const auto running  = [&](auto value) {  // inclusive sums over the places into `weights`, the whole one returned
      u64 v[kEach], s = 0;
#pragma unroll
      for (int q = 0; q < kEach; ++q) {
        const int i = tid * kEach + q;
        s += i < m ? value(i) : 0;
        v[q] = s;
      }
      const u64 incl = warp_scan_u64(s);
      __syncthreads();
      if (lane == 31) warp_part[0][warp] = incl;
      __syncthreads();
      u64 base = incl - s, sum = 0;
      for (int w = 0; w < kWarps; ++w) {
        base += w < warp ? warp_part[0][w] : 0;
        sum += warp_part[0][w];
      }
#pragma unroll
      for (int q = 0; q < kEach; ++q)
        weights[tid * kEach + q] = base + v[q];
      __syncthreads();
      return sum;
    };
    const auto key_at = [&](int i) { return unsigned(list[i] >> 32); };
    u64 total         = running([&](int i) { return key_at(i) >= kmin ? weight(key_at(i)) : 0; });
    if (by_min) {
      u64 left = 0;
      for (int i = tid; i < m; i += kThreads)
        left += key_at(i) >= kmin ? 1 : 0;
      m = int(block_sum(left));
    }
    if (by_p) {
      const u64 of = whole != 0 ? whole : total;
      const double t = ceil(double(top_p) * double(of));
      u64 target     = t >= 1.0 ? u64(t) : 1;
      if (target > of) target = of;
      u64 below = 0;  // places before the one at which the weight reaches the target
      for (int i = tid; i < m; i += kThreads)
        below += weights[i] < target ? 1 : 0;
      below = block_sum(below);
      m     = below + 1 < u64(m) ? int(below) + 1 : m;
      total = weights[m - 1];
    }
    const double t = double(u) * double(total);
    u64 target     = t > 0.0 ? u64(t) : 0;
    if (target >= total) target = total - 1;
    const auto done = [&](int token, unsigned key) {
      write(token, float(log(double(weight(key)) / double(total))));
    };
    if (m <= 128) {  // every place sums the weights of lower tokens itself
      if (tid < m) {
        const u64 mine = list[tid];
        u64 before     = 0;
        for (int i = 0; i < m; ++i) {
          const u64 w = weights[i] - (i > 0 ? weights[i - 1] : 0);
          before += unsigned(list[i]) > unsigned(mine) ? w : 0;  // (the complement of the token)
        }
        const u64 w = weights[tid] - (tid > 0 ? weights[tid - 1] : 0);
        if (before <= target && target < before + w) done(int(0xffffffffu - unsigned(mine)), unsigned(mine >> 32));
      }
      return;
    }
    __syncthreads();
    for (int i = tid; i < m; i += kThreads)
      list[i] = (list[i] << 32) | (list[i] >> 32);  // complements of tokens fall where tokens rise
    __syncthreads();
    sort(m, token_bin);
    (void)running([&](int i) { return weight(unsigned(list[i])); });
    for (int i = tid; i < m; i += kThreads)
      if (weights[i] > target && (i == 0 || weights[i - 1] <= target))
        done(int(0xffffffffu - unsigned(list[i] >> 32)), unsigned(list[i]));
  };
  if (by_k || by_min) {
    const float bound = fmaxf(by_min ? K::value(kmin) : lowest, by_k ? bound_of(u64(top_k)) : lowest);
    const u64* all    = post(count_from(bound));
    u64 n = 0, base = 0;
    for (unsigned r = 0; r < size; ++r) {
      n += all[r];
      base += r < rank ? all[r] : 0;
    }
    if (n <= kList) {
      draw_from_list(bound, int(n), int(base), 0);
      return;
    }
  } else if (by_p) {
    const float bound1 = bound_of(kShort / 2), bound2 = bound_of(kList / 2);
    u64 s[4] = {};  // the whole weight, that of the two beginnings, their lengths
    for (int j = tid; j < part.n; j += kThreads) {
      const Words4 v = raw(j);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float x = K::float_at(v, e);
        const u64 w   = weight_of(x);
        s[0] += w;
        if (x >= bound2) {
          s[2] += w;
          s[3] += u64(1) << 32;
          if (x >= bound1) {
            s[1] += w;
            s[3] += 1;
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      s[q] = warp_sum_u64(s[q]);
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        warp_part[q][warp] = s[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s[q] = 0;
      for (int w = 0; w < kWarps; ++w)
        s[q] += warp_part[q][w];
    }
    const auto all = post4(s);
    u64 ahead      = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s[q] = 0;
      for (unsigned r = 0; r < size; ++r)
        s[q] += all[q][r];
    }
    for (unsigned r = 0; r < rank; ++r)
      ahead += all[3][r];
    const double goal = double(top_p) * double(s[0]);
    const int n1 = int(unsigned(s[3])), n2 = int(s[3] >> 32);
    const bool first = double(s[1]) >= goal && n1 <= kList;
    if (first || (double(s[2]) >= goal && n2 <= kList)) {
      draw_from_list(first ? bound1 : bound2, first ? n1 : n2, first ? int(unsigned(ahead)) : int(ahead >> 32), s[0]);
      return;
    }
  }
  if (by_k) {
    unsigned border;
    u64 above, total;
    if (select(std::true_type{}, weight, [&](u64) { return u64(top_k); }, &border, &above, &total)) {
      tau = border;
      limit_ties(u64(top_k) - above);
    }
  }
  if (by_min && kmin > tau) {
    tau  = kmin;
    last = 0x7fffffff;
  }
  if (by_p) {
    unsigned border;
    u64 above, total, target = 1;
    const auto target_of = [&](u64 whole) {
      const double t = ceil(double(top_p) * double(whole));
      target         = t >= 1.0 ? u64(t) : 1;
      if (target > whole) target = whole;
      return target;
    };
    if (select(std::false_type{}, weight, target_of, &border, &above, &total)) {
      const bool same = border == tau;
      const u64 w     = weight(border);
      tau             = border;
      if (!same) last = 0x7fffffff;
      limit_ties((target - above + w - 1) / w);
    }
  }
  const auto draw_in_place = [&](auto value) {
    u64 before, mine;
    const u64 total = sum_in_order(value, &before, &mine);
    const double t  = double(u) * double(total);
    u64 target      = t > 0.0 ? u64(t) : 0;
    if (target >= total) target = total - 1;  // u of 1 (or more) takes the last kept token
    if (before <= target && target < before + mine && warp == 0) {
      unsigned key;
      const int token = locate(value, target - before, &key);
      if (lane == 0) write(token, float(log(double(weight(key)) / double(total))));
    }
  };
  if (by_k || by_min || by_p) {
    draw_in_place([&](const Words4& v, int e, int token) -> u64 {
      const unsigned key = K::of_bits(K::bits_at(v, e));
      return kept(key, token) ? weight(key) : 0;
    });
  } else {  // (NaN and -inf weigh 0)
    draw_in_place([&](const Words4& v, int e, int) -> u64 { return weight_of(K::float_at(v, e)); });
  }
}

// ---------------------------------------------------------------------------------------
// Host side. The smallest cluster whose parts take at most 64 KB (two CTAs per SM; 256 rows of 131072 bf16 in parts of
// 32 KB and CTAs of 256 threads, three or four per SM, took a tenth longer: more CTAs to a cluster), larger ones while
// there are fewer than two CTAs per SM; parts of up to kMaxPartKb where eight CTAs are not enough, and beyond that rows
// are read from memory in every pass.
// ---------------------------------------------------------------------------------------
template <typename T>
inline cudaError_t launch_sample(Args<T> a, cudaStream_t stream)
{
  constexpr int VE   = Vec16Of<T>::value;
  const int align    = common_alignment({reinterpret_cast<uintptr_t>(a.logits),
                                         a.n_rows > 1 ? uintptr_t(a.ldl) * sizeof(T) : uintptr_t(0)});
  const int64_t most = ceil_div<int64_t>((align >= 16 ? 0 : VE - 1) + int64_t(a.vocab), VE);
  int size           = 1;
  while (size < kMaxCluster && (most > int64_t(size) * 4096 ||
                                (a.n_rows * size < 2 * int64_t(sm_count()) && most > int64_t(size) * 512)))
    size *= 2;
  a.per_cta         = int(ceil_div<int64_t>(most > 0 ? most : 1, size));
  a.shift           = kMaxShift;
  while (a.shift > 0 && (int64_t(1) << (62 - a.shift)) < a.vocab)
    --a.shift;
  const bool cached  = int64_t(a.per_cta) * 16 <= int64_t(kMaxPartKb) * 1024;
  const size_t units = size_t(ceil_div(a.per_cta, 32)) * sizeof(u64);
  const int64_t held = cached ? int64_t(a.per_cta) * 16 : 0;
  a.row_bytes        = int(held > kScratch ? held : kScratch);
  const size_t smem  = size_t(a.row_bytes) + size_t(bins_of(size)) * sizeof(u64) + units;
  const int64_t max_rows = int64_t(0x7fffffff) / size;
  auto kern              = cached ? sample_kernel<T, true> : sample_kernel<T, false>;
  cudaError_t e          = ensure_dynamic_smem(kern, smem);
  if (e != cudaSuccess) return e;
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += max_rows) {
    const int64_t n = a.n_rows - r0 < max_rows ? a.n_rows - r0 : max_rows;
    Args<T> b       = a;
    b.n_rows        = n;
    b.logits += r0 * a.ldl;
    b.uniform += r0;
    if (b.temperature) b.temperature += r0;
    if (b.top_k) b.top_k += r0;
    if (b.top_p) b.top_p += r0;
    if (b.min_p) b.min_p += r0;
    if (b.logprobs) b.logprobs += r0;
    b.out = static_cast<char*>(a.out) + r0 * (a.out64 ? 8 : 4);
    e     = distill::launch_clusters(kern, b, n * size, size, kThreads, smem, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace sample
}  // namespace detail
}  // namespace raft_b200
