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
// most kMaxShift (45 bits for 131072 tokens): exact, the same whatever the order, the split of the row or the number of rows of the call.
//
// A cluster of CTAs takes a row, every CTA a part, which it keeps in shared memory. The logits' bits, made to rise with
// their value, are counted by their first kDigitBits as soon as the row has come in, and the counts bound the beginning
// of the order that can be kept: by top_k, by the bin of the lowest logit that min_p admits, or, for a top-p alone, by
// taking a beginning of at most kShort or kList tokens and looking whether its weight is enough. It is collected in the
// first CTA, sorted, and the rest happens there; the others are done. Longer beginnings (a flat distribution, a large k)
// are narrowed by radix selection, a digit at a time, by counts or weights summed over the cluster through distributed
// shared memory, and drawn from in place.
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
constexpr int kShort      = 512;  // sorted by counting, a token per thread
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
B2R_DI unsigned cluster_fetch_add_u32(unsigned* p, unsigned rank, unsigned v)
{
  unsigned old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;"
               : "=r"(old)
               : "r"(cluster_address(p, rank)), "r"(v)
               : "memory");
  return old;
}
B2R_DI void cluster_sync()
{
  distill::cluster_arrive();
  distill::cluster_wait();
}

template <typename T, bool kCached>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  using K          = Key<T>;
  extern __shared__ __align__(16) unsigned char sample_smem[];
  __shared__ __align__(16) unsigned hist[2][kBins];           // counts of this CTA; low and high words of the bins' sums
  __shared__ __align__(16) unsigned totals[kBins];            // counts of the row
  __shared__ __align__(16) u64 bins[kBins];     // sums over the cluster of the bins this CTA looks after
  __shared__ double powers[32];                 // 2^(i / 32)
  __shared__ unsigned kmax_all, list_n, list_at, list_base;
  __shared__ u64 posted[4][3][kMaxCluster];     // up to three values of every CTA, four exchanges deep
  __shared__ u64 result[2][2];
  __shared__ u64 warp_part[3][kWarps];
  __shared__ u64 carry;
  Words4* slice = reinterpret_cast<Words4*>(sample_smem);  // [per_cta] if kCached
  u64* units    = reinterpret_cast<u64*>(slice + (kCached ? a.per_cta : 0));  // sums of 32 vectors each, in order
  const unsigned rank = distill::cluster_rank();
  const unsigned size = distill::cluster_size();
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
  if (tid == 0) kmax_all = list_n = list_at = 0;
  __syncthreads();
  distill::cluster_arrive();  // every CTA of the cluster has started and is set up
  const float temp   = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  const int top_k    = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  const float top_p  = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  const float min_p  = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  const float u      = a.uniform[row];
  const bool greedy  = !(temp > 0.0f);
  const auto vec     = [&](int j) { return kCached ? slice[j] : K::pack(part.load(j)); };  // keys
  int exchanges      = 0;

  // every CTA's values, known to all afterwards (four calls long)
  auto post3 = [&](u64 v0, u64 v1, u64 v2) {
    auto slot = posted[exchanges & 3];
    ++exchanges;
    if (tid < int(size)) {
      cluster_store_u64(&slot[0][rank], unsigned(tid), v0);
      cluster_store_u64(&slot[1][rank], unsigned(tid), v1);
      cluster_store_u64(&slot[2][rank], unsigned(tid), v2);
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

  // the row, its largest key, and (where anything is to be left out) the counts by the first digit
  const bool by_k    = !greedy && top_k > 0 && top_k < a.vocab;
  const bool by_p    = !greedy && top_p < 1.0f;
  const bool by_min  = !greedy && min_p > 0.0f;
  const bool counted = by_k || by_p || by_min;
  constexpr int kLow = K::kBits - kDigitBits;  // bits behind the first digit
  unsigned kmax      = 0;
  if constexpr (kCached) distill::copy_wait<0>();
  for (int j = tid; j < part.n; j += kThreads) {
    const Words4 v = K::pack(kCached ? slice[j] : part.load(j));
    if (kCached) slice[j] = v;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const unsigned key = K::at(v, e);
      kmax               = max(kmax, key);
      if (counted && key > K::kNegInf) atomicAdd(&hist[0][key >> kLow], 1u);
    }
  }
  kmax = __reduce_max_sync(distill::kFull, kmax);
  __syncthreads();
  distill::cluster_wait();
  if (lane < int(size)) cluster_max_u32(&kmax_all, unsigned(lane), kmax);
  if (counted) {
    for (int i = tid; i < kBins; i += kThreads) {
      const unsigned n = hist[0][i];
      if (n != 0)
        for (unsigned r = 0; r < size; ++r)
          cluster_add_u32(&totals[i], r, n);
    }
  }
  cluster_sync();
  kmax = kmax_all;
  auto write = [&](int64_t token, float logprob) {  // by one thread of the cluster
    if (a.out64)
      static_cast<long long*>(a.out)[row] = token;
    else
      static_cast<int*>(a.out)[row] = int(token);
    if (a.logprobs != nullptr) a.logprobs[row] = logprob;
  };
  if (kmax <= K::kNegInf) {  // nothing to draw from
    if (rank == 0 && tid == 0) write(-1, -INFINITY);
    return;
  }
  // 2^x by table and polynomial: x * 32 = n + r, 2^x = 2^(n / 32) 2^(r / 32), the second by its Taylor series to the
  // fifth power (|r / 32| <= 1 / 64: 3e-15), the first from `powers` and an exponent (P. T. P. Tang, 1989). What rounds
  // to 0 is cut off at `low` (and NaN there is none); temperatures above 1e30 count as that.
  const double zmax    = double(K::value(kmax));
  const double slope   = 1.4426950408889634 / double(fminf(temp, 1e30f));
  const double slope32 = slope * 32.0;
  const int shift      = a.shift;
  const bool infinite  = kmax == K::kZero + (K::kZero - K::kNegInf);  // a +inf logit: the others weigh nothing
  const float low      = fmaxf(__double2float_rd(zmax - double(shift + 2) / slope), -FLT_MAX);
  const auto weight    = [&](unsigned key) -> u64 {
    const double y   = (double(fmaxf(K::value(key), low)) - zmax) * slope32;
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
    return !infinite ? whole : (key == kmax ? u64(1) << shift : 0);
  };

  // kept: key > tau, or key == tau and token <= last
  unsigned tau = K::kNegInf + 1;
  int last     = 0x7fffffff;
  const auto kept = [&](unsigned key, int token) { return key > tau || (key == tau && token <= last); };

  // Sums of value(key, token) over runs of 32 vectors; *before: of the CTAs ahead of this one. Returns the whole sum.
  auto sum_in_order = [&](auto value, u64* before, u64* mine) {
    u64 own = 0;
    for (int j0 = warp * 32; j0 < part.n; j0 += kThreads) {
      u64 s = 0;
      if (j0 + lane < part.n) {
        const Words4 v = vec(j0 + lane);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          s += value(K::at(v, e), part.first + (j0 + lane) * VE + e);
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
    Words4 v    = K::pack(distill::minus_inf<T>());
    u64 s       = 0;
    if (j < part.n) {
      v = vec(j);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        s += value(K::at(v, e), part.first + j * VE + e);
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
      upto += value(K::at(v, e), t);
      if (token < 0 && upto > target) {
        token = t;
        found = K::at(v, e);
      }
    }
    *key = __shfl_sync(distill::kFull, found, l);
    return __shfl_sync(distill::kFull, token, l);
  };
  // The border of the order at which the sum of value(key) over the kept tokens reaches `target` (at least 1, at most
  // the whole sum): its key in *border, the sum over larger keys in *above. With kCount the values are 1.
  // A target above the whole sum, which is returned in *total: the border is below every kept key, false. With fewer
  // `digits` than keys have, the border's first ones.
  auto select = [&](auto count, auto value, auto target_of, int digits, unsigned* border, u64* above, u64* total) {
    constexpr bool kCount = decltype(count)::value;
    unsigned prefix = 0;  // bits of the border found so far
    int left        = K::kBits;
    u64 over        = 0;
    u64 target      = 0;
    while (left > 0 && digits-- > 0) {
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
    const auto is_tie = [&](unsigned key, int token) -> u64 { return key == tau && token <= last ? 1 : 0; };
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

  if (greedy) {
    tau = kmax;
    const auto is_max = [&](unsigned key, int) -> u64 { return key == kmax ? 1 : 0; };
    u64 before, mine;
    (void)sum_in_order(is_max, &before, &mine);
    if (before == 0 && mine > 0 && warp == 0) {
      unsigned key;
      const int token = locate(is_max, 0, &key);
      if (lane == 0) write(token, 0.0f);
    }
    return;
  }
  // The lowest bin of the first digit that can hold kept tokens, and the number of tokens from it up.
  // w >= min_p, as a bound on the key
  const double mp     = min_p < 1.0f ? double(min_p) : 1.0;
  const unsigned kmin = !by_min ? 0u : (mp == 1.0 ? kmax : min(kmax, K::at_least(zmax + log2(mp) / slope)));
  // tokens of the bins from `bin` up: of the row in the high word, of this CTA in the low one
  const auto tokens_from = [&](unsigned bin) {
    u64 s = 0;
    for (int i = tid; i < kBins; i += kThreads)
      if (unsigned(i) >= bin) s += (u64(totals[i]) << 32) | hist[0][i];
    return block_sum(s);
  };
  // The largest bin from which up there are at least `goal` tokens (0: there are fewer in all).
  const auto bin_of = [&](u64 goal) {
    constexpr int kEach = kBins / kThreads;
    const int top       = kBins - 1 - tid * kEach;
    u64 s               = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q)
      s += totals[top - q];
    const u64 incl = warp_scan_u64(s);
    __syncthreads();
    if (lane == 31) warp_part[0][warp] = incl;
    if (tid == 0) carry = 0;
    __syncthreads();
    u64 run = incl - s;
    for (int w = 0; w < warp; ++w)
      run += warp_part[0][w];
    if (run < goal && goal <= run + s) {
      int q = 0;
      while ((run += totals[top - q]) < goal)
        ++q;
      carry = u64(top - q);
    }
    __syncthreads();
    return unsigned(carry);
  };
  // Draws from the tokens of the bins from `bin` up, all of whose n are collected in the first CTA. `whole`: the weight
  // of all tokens that top-p is measured by, or 0: that of the first top_k and min-p leave. `own` of them are here.
  auto draw_from_list = [&](unsigned bin, int n, unsigned own, u64 whole) {
    if (tid == 0) list_base = cluster_fetch_add_u32(&list_n, 0, own);
    __syncthreads();
    for (int j = tid; j < part.n && own != 0; j += kThreads) {
      const Words4 v = vec(j);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const unsigned key = K::at(v, e);
        if (key > K::kNegInf && (key >> kLow) >= bin) {
          const unsigned token = unsigned(part.first + j * VE + e);
          // larger keys first, lower tokens first among equals
          cluster_store_u64(&bins[list_base + atomicAdd(&list_at, 1u)], 0, (u64(key) << 32) | (0xffffffffu - token));
        }
      }
    }
    cluster_sync();
    if (rank != 0) return;
    u64* list    = bins;
    u64* weights = reinterpret_cast<u64*>(&hist[0][0]);  // [kList]
    // falling order of list[0 .. n)
    const auto sort = [&](int count) {
      if (count <= kShort) {  // a thread's place is the number of larger ones; no two are equal
        __syncthreads();
        const u64 mine = tid < count ? list[tid] : 0;
        if (tid >= count && tid < (count + 1) / 2 * 2) list[tid] = 0;
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
      int padded = 32;
      while (padded < count)
        padded *= 2;
      for (int i = count + tid; i < padded; i += kThreads)
        list[i] = 0;
      for (int k = 2; k <= padded; k *= 2) {
        for (int h = k / 2; h > 0; h /= 2) {
          __syncthreads();
          for (int i = tid; i < padded / 2; i += kThreads) {
            const int lo = 2 * i - (i & (h - 1)), hi = lo + h;
            const u64 x = list[lo], y = list[hi];
            if ((x < y) == ((lo & k) == 0)) {
              list[lo] = y;
              list[hi] = x;
            }
          }
        }
      }
      __syncthreads();
    };
    sort(n);
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
    sort(m);
    (void)running([&](int i) { return weight(unsigned(list[i])); });
    for (int i = tid; i < m; i += kThreads)
      if (weights[i] > target && (i == 0 || weights[i - 1] <= target))
        done(int(0xffffffffu - unsigned(list[i] >> 32)), unsigned(list[i]));
  };
  if (by_k || by_min) {
    const unsigned bin = max(kmin >> kLow, by_k ? bin_of(u64(top_k)) : 0u);
    const u64 n        = tokens_from(bin);
    if ((n >> 32) <= kList) {
      draw_from_list(bin, int(n >> 32), unsigned(n), 0);
      return;
    }
  } else if (by_p) {
    // beginnings of at most kShort and kList tokens, and their weights
    const unsigned bin1 = bin_of(kShort + 1) + 1, bin2 = bin_of(kList + 1) + 1;
    u64 s0 = 0, s1 = 0, s2 = 0;
    for (int j = tid; j < part.n; j += kThreads) {
      const Words4 v = vec(j);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const unsigned key = K::at(v, e);
        const u64 w        = key > K::kNegInf ? weight(key) : 0;
        s0 += w;
        s1 += (key >> kLow) >= bin1 ? w : 0;
        s2 += (key >> kLow) >= bin2 ? w : 0;
      }
    }
    s0 = warp_sum_u64(s0);
    s1 = warp_sum_u64(s1);
    s2 = warp_sum_u64(s2);
    __syncthreads();
    if (lane == 0) {
      warp_part[0][warp] = s0;
      warp_part[1][warp] = s1;
      warp_part[2][warp] = s2;
    }
    __syncthreads();
    s0 = s1 = s2 = 0;
    for (int w = 0; w < kWarps; ++w) {
      s0 += warp_part[0][w];
      s1 += warp_part[1][w];
      s2 += warp_part[2][w];
    }
    const auto all = post3(s0, s1, s2);
    s0 = s1 = s2 = 0;
    for (unsigned r = 0; r < size; ++r) {
      s0 += all[0][r];
      s1 += all[1][r];
      s2 += all[2][r];
    }
    const double goal = double(top_p) * double(s0);
    if (double(s2) >= goal && s2 > 0) {
      const unsigned bin = double(s1) >= goal && s1 > 0 ? bin1 : bin2;
      const u64 n        = tokens_from(bin);
      draw_from_list(bin, int(n >> 32), unsigned(n), s0);
      return;
    }
  }
  if (by_k) {
    unsigned border;
    u64 above, total;
    if (select(std::true_type{}, weight, [&](u64) { return u64(top_k); }, 4, &border, &above, &total)) {
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
    if (select(std::false_type{}, weight, target_of, 4, &border, &above, &total)) {
      const bool same = border == tau;
      const u64 w     = weight(border);
      tau             = border;
      if (!same) last = 0x7fffffff;
      limit_ties((target - above + w - 1) / w);
    }
  }
  const auto kept_weight = [&](unsigned key, int token) -> u64 { return kept(key, token) ? weight(key) : 0; };
  u64 before, mine;
  const u64 total = sum_in_order(kept_weight, &before, &mine);
  const double t  = double(u) * double(total);
  u64 target      = t > 0.0 ? u64(t) : 0;
  if (target >= total) target = total - 1;  // u of 1 (or more) takes the last kept token
  if (before <= target && target < before + mine && warp == 0) {
    unsigned key;
    const int token = locate(kept_weight, target - before, &key);
    if (lane == 0) write(token, float(log(double(weight(key)) / double(total))));
  }
}

// ---------------------------------------------------------------------------------------
// Host side. The smallest cluster whose parts take at most 64 KB (three CTAs per SM), larger ones while there are
// fewer than two CTAs per SM; parts of up to kMaxPartKb where eight CTAs are not enough, and beyond that rows are read
// from memory in every pass.
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
  const size_t smem  = (cached ? size_t(a.per_cta) * 16 : 0) + units;
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
