// Distillation from a teacher's top logits.
//
// A row has student logits z over the vocabulary and a list of (token, teacher logit) pairs. With the temperature T
//     p = softmax(teacher / T) over the valid entries of the list         (token in [0, vocab))
//     q = softmax(z / T)       over the vocabulary
//     loss = T^2 * sum_k p_k (log p_k - log q[id_k]),     lse = log sum_v exp(z_v / T)
//     d loss / d z_v = T (q_v - sum of p_k with id_k = v)
// A row without a valid entry (all tokens -1: prompt or padding positions) has loss 0 and gradient 0.
//
// The pass over the logits is what costs: V elements per row are read once, and written once where the gradient is
// wanted. For the gradient a row is spread over the CTAs of a cluster, which keep its exponentials in registers
// between the two uses, so that no second read is needed; the CTAs exchange (maximum, sum) pairs through distributed
// shared memory. Sums and statistics are fp32, relative to the maximum; the loss, a sum of k terms, is fp64.
#pragma once

#include "launch.cuh"
#include "vocab_common.cuh"

#include <cfloat>

namespace raft_b200 {
namespace detail {
namespace distill {

constexpr int kMaxK      = 1024;
constexpr unsigned kFull = 0xffffffffu;

// ids and teacher logits of a list: types are looked up per entry (a list is short)
struct List {
  const void* ids;
  int64_t ldi;
  const void* teacher;
  int64_t ldt;
  int id64;  // tokens are int64 (else int32)
  int tdt;   // b2r_dtype of the teacher's logits
  int k;

  B2R_DI int64_t id(int64_t row, int j) const
  {
    return id64 ? int64_t(static_cast<const long long*>(ids)[row * ldi + j])
                : int64_t(static_cast<const int*>(ids)[row * ldi + j]);
  }
  B2R_DI float logit(int64_t row, int j) const
  {
    const int64_t at = row * ldt + j;
    if (tdt == 2) return __half2float(static_cast<const __half*>(teacher)[at]);               // B2R_F16
    if (tdt == 7) return __bfloat162float(static_cast<const __nv_bfloat16*>(teacher)[at]);    // B2R_BF16
    return static_cast<const float*>(teacher)[at];
  }
};

template <typename T>
struct Args {
  const T* logits;
  int64_t ldl;
  T* grad;  // null: loss only
  int64_t ldg;
  float* loss;  // each may be null
  float* lse;
  const float* grad_loss;
  const float* lse_in;  // gradient alone: the forward pass's lse
  List list;
  int64_t n_rows;
  int vocab;
  double temperature;
  int per_cta;  // vectors of a row per CTA of the cluster
};

B2R_DI float ex2(float x)
{
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

B2R_DI unsigned cluster_rank()
{
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
B2R_DI unsigned cluster_size()
{
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
B2R_DI void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
B2R_DI void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// v to the float2 at the same shared-memory address in CTA `rank` of the cluster
B2R_DI void cluster_store(float2* p, unsigned rank, float2 v)
{
  const unsigned local = unsigned(__cvta_generic_to_shared(p));
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}

B2R_DI void cluster_store_f64(double* p, unsigned rank, double v)
{
  const unsigned local = unsigned(__cvta_generic_to_shared(p));
  unsigned remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(v) : "memory");
}

// One row as 16-byte vectors of its memory: vector j holds elements [j * VE - phase, (j + 1) * VE - phase), where
// `phase` elements lie between the 16-byte boundary at or before the row's first element and that element. Only
// whole vectors are moved as vectors; the elements of the first and last one are moved one by one, so nothing
// outside the row is touched.
template <typename T>
struct RowVecs {
  static constexpr int VE = Vec16Of<T>::value;
  int phase, vocab, n;  // n vectors

  B2R_DI RowVecs(const T* row, int v)
  {
    phase = int((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    vocab = v;
    n     = (phase + v + VE - 1) / VE;
  }
  B2R_DI int first(int j) const { return j * VE - phase; }  // element index of lane 0 of vector j
  B2R_DI bool whole(int j) const { return first(j) >= 0 && first(j) + VE <= vocab; }

  B2R_DI VecOf<T, VE> load(const T* row, int j) const
  {
    VecOf<T, VE> r;
    if (j < n && whole(j)) {
      uint32_t w[4];  // not the non-coherent path: the gradient may be written over the logits
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(row + first(j))
                   : "memory");
      memcpy(&r, w, 16);
      return r;
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int e = first(j) + i;
      r.e[i]      = j < n && e >= 0 && e < vocab ? row[e] : FloatIo<T>::down(-INFINITY);
    }
    return r;
  }
  // `same`: the row of `dst` has the same phase
  B2R_DI void store(T* dst, int j, const VecOf<T, VE>& v, bool same) const
  {
    if (j >= n) return;
    if (same && whole(j)) {
      store_vec<T, VE>(dst + first(j), v);
      return;
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int e = first(j) + i;
      if (e >= 0 && e < vocab) dst[e] = v.e[i];
    }
  }
};

// 16 bytes from global to shared memory, asynchronous (the thread's own commit / wait groups order it)
B2R_DI void copy_async16(void* smem, const void* g)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(unsigned(__cvta_generic_to_shared(smem))), "l"(g)
               : "memory");
}
B2R_DI void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
B2R_DI void copy_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

B2R_DI float warp_max(float v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <typename F>
B2R_DI F warp_sum(F v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// sum_v 2^(c z_v) as s * 2^(c m): m the largest logit, s relative to it (m = -inf: nothing seen but -inf; s is 0
// then, or NaN). Exponents are always formed from DIFFERENCES of logits: c * m can overflow (a row at the type's
// lowest value), and a difference near the maximum is exact, so no rounding scales a whole row.
struct ExpSum {
  float m, s;
};
B2R_DI ExpSum warp_join(ExpSum v, float c)
{
  const float m = warp_max(v.m);
  return {m, warp_sum(v.m == -INFINITY ? v.s : v.s * ex2((v.m - m) * c))};
}
// every warp's (m, s) of a cluster, the same result in every lane
B2R_DI ExpSum join_parts(const float2* parts, int n, float c)
{
  ExpSum all = {-INFINITY, 0.0f};
  for (int i = int(threadIdx.x) & 31; i < n; i += 32) {
    const float2 v = parts[i];
    const float m  = fmaxf(all.m, v.x);
    all.s          = (all.m == -INFINITY ? all.s : all.s * ex2((all.m - m) * c)) +
            (v.x == -INFINITY ? v.y : v.y * ex2((v.x - m) * c));
    all.m = m;
  }
  return warp_join(all, c);
}

// The list in shared memory, an entry per place: token (-1: not valid) and teacher logit, then log weight. One warp
// turns the logits into log weights; returns whether any entry is valid. Places of the list are spread over lanes the
// same way in every loop, so a lane meets only what it wrote itself.
B2R_DI bool weigh_list(const int* id, float* y, int k, float inv_t)
{
  const int lane = int(threadIdx.x) & 31;
  float m        = -INFINITY;
  bool nan       = false;
  for (int j = lane; j < k; j += 32) {
    if (id[j] < 0) continue;
    m   = fmaxf(m, y[j]);
    nan = nan || y[j] != y[j];
  }
  m               = warp_max(m);
  nan             = __any_sync(kFull, nan);
  const bool some = m > -INFINITY || nan;
  float s         = 0.0f;
  for (int j = lane; j < k; j += 32)
    s += some && id[j] >= 0 ? expf((y[j] - m) * inv_t) : 0.0f;
  const float ls = logf(warp_sum(s));
  for (int j = lane; j < k; j += 32)
    y[j] = some && id[j] >= 0 ? (y[j] - m) * inv_t - ls : -INFINITY;
  return some;
}

// Entry j of a row's list as weigh_list wants it.
template <typename T>
B2R_DI void fetch_entry(const Args<T>& a, int64_t row, int j, int* id, float* y)
{
  const int64_t t = a.list.id(row, j);
  const bool ok   = t >= 0 && t < a.vocab;
  *id             = ok ? int(t) : -1;
  *y              = ok ? a.list.logit(row, j) : -INFINITY;
}

// Weight of entry j's token over the whole list (a token may be named more than once); false unless j is the first
// entry of its token, which speaks for all of them.
B2R_DI bool listed_weight(const int* id, const float* logp, int k, int j, float* w)
{
  const int t = id[j];
  float sum   = 0.0f;
  bool first  = true;
  for (int i = 0; i < k; ++i) {
    if (id[i] == t) {
      first = first && i >= j;
      sum += expf(logp[i]);
    }
  }
  *w = sum;
  return first;
}

// ---------------------------------------------------------------------------------------
// Loss and gradient in one pass. A cluster takes a row, every CTA of it `per_cta` vectors; clusters are persistent and
// walk the rows. Every thread copies its own vectors of the rows to come into shared memory (two rows ahead, kStages
// buffers), so that the memory system is busy while a row is worked on, and nobody has to wait for anybody to use
// them. A thread turns its elements into exponentials relative to its own maximum and keeps those in registers; ONE
// cluster barrier per row carries the (m, s) of every warp to every CTA, after which the gradient is a product per
// element. One exponential per element: at two the MUFU unit (16 per clock and SM) would bound the kernel.
//
// Everything that hangs on the list runs beside that, a step ahead or behind, so that its chains of dependent loads
// are off the path: entries are loaded two rows ahead, their softmax is taken one row ahead by one warp, the student
// logits of listed tokens are read from the buffers of the CTA that holds them, and the listed elements of the
// gradient are written one barrier after the vectors they lie in (the barrier orders the two writes).
// ---------------------------------------------------------------------------------------
constexpr int kStages = 3;
constexpr int kStepNv = 4;

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
distill_step_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  constexpr int NV = kStepNv;
  constexpr int NW = NT / 32;
  using Vec        = VecOf<T, VE>;
  extern __shared__ __align__(16) unsigned char step_smem[];
  __shared__ float2 parts[2][8 * NW];   // (m, s) of every warp of the cluster, by CTA rank
  __shared__ double loss_part[2][8];    // rank 0: the loss sums of the CTAs
  __shared__ int some_s[3];
  Vec* stages   = reinterpret_cast<Vec*>(step_smem);             // [kStages][NT * NV]
  const int k   = a.list.k;
  int* ids      = reinterpret_cast<int*>(stages + kStages * NT * NV);  // [3][k]
  float* logps  = reinterpret_cast<float*>(ids + 3 * k);               // [3][k]
  int* late_id  = reinterpret_cast<int*>(logps + 3 * k);               // [k] token whose element is still to be written
  float* late_v = reinterpret_cast<float*>(late_id + k);               // [k]
  const unsigned rank = cluster_rank();
  const unsigned size = cluster_size();
  const int tid       = int(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31;
  cluster_arrive();  // every CTA of the cluster has started: waited for before the first remote store
  grid_dep_sync();

  const int64_t step  = int64_t(gridDim.x) / size;
  const int64_t first = int64_t(blockIdx.x) / size;
  const float c       = float(1.4426950408889634 / a.temperature);
  const float inv_t   = float(1.0 / a.temperature);
  const int j0        = int(rank) * a.per_cta;

  // the thread's vectors of a row on their way into buffer `stage`
  auto request = [&](int64_t row, int stage) {
    if (row < a.n_rows) {
      const T* z = a.logits + row * a.ldl;
      const RowVecs<T> rv(z, a.vocab);
      const int j1 = j0 + a.per_cta < rv.n ? j0 + a.per_cta : rv.n;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = j0 + i * NT + tid;
        if (j < j1) {
          Vec* to = stages + stage * (NT * NV) + i * NT + tid;
          if (rv.whole(j))
            copy_async16(to, z + rv.first(j));
          else
            *to = rv.load(z, j);
        }
      }
    }
    copy_commit();
  };
  // entry `tid` of a row's list in registers (lists longer than the CTA: the rest is fetched where it is stored)
  int next_id  = -1;
  float next_y = 0.0f;
  auto ask_list = [&](int64_t row) {
    if (row < a.n_rows && tid < k) fetch_entry(a, row, tid, &next_id, &next_y);
  };
  auto store_list = [&](int64_t row, int buf) {
    if (row >= a.n_rows) return;
    if (tid < k) {
      ids[buf * k + tid]   = next_id;
      logps[buf * k + tid] = next_y;
    }
    for (int j = tid + NT; j < k; j += NT)
      fetch_entry(a, row, j, &ids[buf * k + j], &logps[buf * k + j]);
  };
  for (int j = tid; j < k; j += NT)
    late_id[j] = -1;

  request(first, 0);
  request(first + step, 1);
  ask_list(first);
  store_list(first, 0);
  ask_list(first + step);
  __syncthreads();
  if (warp == NW - 1 && first < a.n_rows) {
    const bool some = weigh_list(ids, logps, k, inv_t);
    if (lane == 0) some_s[0] = some;
  }
  cluster_wait();

  int64_t late_row = -1;  // row whose listed elements and loss are still to be written
  int stage        = 0;   // it % kStages == it % 3: buffer of the row's vectors and of its list
  double my_loss   = 0.0;
  float late_lse   = 0.0f;
  int par          = 0;   // it & 1
  for (int64_t row = first;; row += step, par ^= 1) {
    const bool on       = row < a.n_rows;  // the last turn only finishes what is late
    const int stage1    = stage + 1 == kStages ? 0 : stage + 1;
    const T* z          = a.logits + (on ? row : 0) * a.ldl;
    const RowVecs<T> rv(z, a.vocab);
    const int j1        = j0 + a.per_cta < rv.n ? j0 + a.per_cta : rv.n;
    store_list(row + step, stage1);
    ask_list(row + 2 * step);
    const Vec* mine = stages + stage * (NT * NV) + tid;
    float e[NV * VE];
    float m = -INFINITY;
    if (on) {
      copy_wait<1>();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (j0 + i * NT + tid < j1) {
          const Vec v = mine[i * NT];
#pragma unroll
          for (int q = 0; q < VE; ++q) {
            e[i * VE + q] = FloatIo<T>::up(v.e[q]);
            m             = fmaxf(m, e[i * VE + q]);
          }
        } else {
#pragma unroll
          for (int q = 0; q < VE; ++q)
            e[i * VE + q] = -INFINITY;
        }
      }
      const float base = m == -INFINITY ? 0.0f : m;
      float s          = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (j0 + i * NT < j1) {
#pragma unroll
          for (int q = 0; q < VE; ++q) {
            e[i * VE + q] = ex2((e[i * VE + q] - base) * c);
            s += e[i * VE + q];
          }
        }
      }
      const ExpSum w = warp_join({m, s}, c);
      if (lane < int(size)) cluster_store(&parts[par][rank * NW + warp], unsigned(lane), make_float2(w.m, w.s));
    }
    if (late_row >= 0 && warp == 0 && lane == 0) cluster_store_f64(&loss_part[par][rank], 0, my_loss);
    cluster_arrive();
    cluster_wait();

    if (late_row >= 0) {
      T* g = a.grad + late_row * a.ldg;
      for (int j = tid; j < k; j += NT) {
        if (late_id[j] >= 0) g[late_id[j]] = FloatIo<T>::down(late_v[j]);
        late_id[j] = -1;
      }
      if (rank == 0 && tid == 0) {
        double sum = 0.0;
        for (unsigned r = 0; r < size; ++r)
          sum += loss_part[par][r];
        if (a.loss != nullptr) a.loss[late_row] = float(sum * a.temperature * a.temperature);
        if (a.lse != nullptr) a.lse[late_row] = late_lse;
      }
    }
    if (!on) break;
    request(row + 2 * step, stage == 0 ? kStages - 1 : stage - 1);

    const ExpSum all   = join_parts(parts[par], int(size) * NW, c);
    const float l2s    = log2f(all.s);
    const bool some    = some_s[stage] != 0;
    const float factor = some ? float(double(a.grad_loss[row]) * a.temperature) : 0.0f;
    // a thread without a maximum holds zeros (or NaN)
    const float scale = (m == -INFINITY ? (all.s > 0.0f ? 0.0f : NAN) : ex2((m - all.m) * c - l2s)) * factor;
    T* g               = a.grad + row * a.ldg;
    const bool same    = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = j0 + i * NT + tid;
      if (j < j1) {
        Vec o;
#pragma unroll
        for (int q = 0; q < VE; ++q)
          o.e[q] = FloatIo<T>::down(some ? e[i * VE + q] * scale : 0.0f);
        rv.store(g, j, o, same);
      }
    }
    // the list's part
    const int* id     = ids + stage * k;
    const float* logp = logps + stage * k;
    const T* held     = reinterpret_cast<const T*>(stages + stage * (NT * NV)) - rv.first(j0);  // held[t]: token t
    const int lo      = rv.first(j0) > 0 ? rv.first(j0) : 0;
    const int hi      = rv.first(j1) < a.vocab ? rv.first(j1) : a.vocab;
    if (some) {
      for (int j = tid; j < k; j += NT) {
        const int t = id[j];
        float w;
        if (t >= lo && t < hi && listed_weight(id, logp, k, j, &w)) {
          late_id[j] = t;
          late_v[j]  = factor * (ex2((FloatIo<T>::up(held[t]) - all.m) * c - l2s) - w);
        }
      }
    }
    if (warp == 0) {
      const double lse = double(all.m) / a.temperature + double(logf(all.s));
      double sum       = 0.0;
      for (int j = lane; j < k && some; j += 32) {
        const int t    = id[j];
        const float lp = logp[j];
        if (t >= lo && t < hi && !(lp == -INFINITY))
          sum += double(expf(lp)) * (double(lp) - (double(FloatIo<T>::up(held[t])) / a.temperature - lse));
      }
      my_loss  = warp_sum(sum);
      late_lse = float(lse);
    }
    if (warp == NW - 1 && row + step < a.n_rows) {
      const bool next = weigh_list(ids + stage1 * k, logps + stage1 * k, k, inv_t);
      if (lane == 0) some_s[stage1] = next;
    }
    late_row = row;
    stage    = stage1;
  }
  copy_wait<0>();
}

// ---------------------------------------------------------------------------------------
// Rows that do not fit the registers of a cluster (kGrad), and the loss alone: NT threads stream their CTA's part of
// the row, the next vectors under way while these are worked on, and one more warp of rank 0's CTA takes the list.
// With kGrad every part is read a second time.
// ---------------------------------------------------------------------------------------
constexpr int kStreamNv = 4;

template <typename T, int NT, bool kGrad>
__global__ void __launch_bounds__(NT + 32)
distill_stream_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  constexpr int NV = kStreamNv;
  constexpr int NW = NT / 32;
  using Vec        = VecOf<T, VE>;
  extern __shared__ __align__(16) unsigned char stream_smem[];
  __shared__ float2 parts[8 * NW];
  __shared__ int some_s;
  const unsigned rank = cluster_rank();
  const unsigned size = cluster_size();
  const int tid       = int(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31;
  const int k   = a.list.k;
  int* id       = reinterpret_cast<int*>(stream_smem);  // [k]
  float* logp   = reinterpret_cast<float*>(id + k);     // [k]
  float* zid    = logp + k;                             // [k] student logits of the listed tokens
  cluster_arrive();
  grid_dep_sync();
  const int64_t row = int64_t(blockIdx.x) / size;
  const T* z        = a.logits + row * a.ldl;
  const RowVecs<T> rv(z, a.vocab);
  const int j0  = int(rank) * a.per_cta;
  const int j1  = j0 + a.per_cta < rv.n ? j0 + a.per_cta : rv.n;
  const float c = float(1.4426950408889634 / a.temperature);
  if (warp == NW) {  // the list
    if (kGrad || rank == 0) {
      for (int j = lane; j < k; j += 32) {
        fetch_entry(a, row, j, &id[j], &logp[j]);
        zid[j] = id[j] >= 0 ? FloatIo<T>::up(z[id[j]]) : 0.0f;
      }
      const bool some = weigh_list(id, logp, k, float(1.0 / a.temperature));
      if (lane == 0) some_s = some;
    }
    cluster_wait();
  } else {
    float m = -INFINITY, s = 0.0f;  // as ExpSum
    Vec cur[NV], nxt[NV];
    auto fetch = [&](Vec(&v)[NV], int j) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int q = j + i * NT + tid;
        if (q < j1) v[i] = rv.load(z, q);
      }
    };
    auto use = [&](const Vec(&v)[NV], int j) {
      float top = m;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (j + i * NT + tid < j1) {
#pragma unroll
          for (int q = 0; q < VE; ++q)
            top = fmaxf(top, FloatIo<T>::up(v[i].e[q]));
        }
      }
      if (top > m) {
        s = m == -INFINITY ? s : s * ex2((m - top) * c);
        m = top;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (j + i * NT + tid < j1) {
#pragma unroll
          for (int q = 0; q < VE; ++q)
            s += ex2((FloatIo<T>::up(v[i].e[q]) - base) * c);
        }
      }
    };
    fetch(cur, j0);
    for (int j = j0; j < j1; j += 2 * NV * NT) {
      fetch(nxt, j + NV * NT);
      use(cur, j);
      fetch(cur, j + 2 * NV * NT);
      use(nxt, j + NV * NT);
    }
    const ExpSum w = warp_join({m, s}, c);
    cluster_wait();
    if (lane < int(size)) cluster_store(&parts[rank * NW + warp], unsigned(lane), make_float2(w.m, w.s));
  }
  cluster_arrive();
  cluster_wait();
  const ExpSum all = join_parts(parts, int(size) * NW, c);
  if (rank == 0 && warp == NW) {
    const bool some  = some_s != 0;
    const double lse = double(all.m) / a.temperature + double(logf(all.s));
    double sum       = 0.0;
    for (int j = lane; j < k && some; j += 32) {
      if (id[j] >= 0 && !(logp[j] == -INFINITY))
        sum += double(expf(logp[j])) * (double(logp[j]) - (double(zid[j]) / a.temperature - lse));
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      if (a.loss != nullptr) a.loss[row] = float(sum * a.temperature * a.temperature);
      if (a.lse != nullptr) a.lse[row] = float(lse);
    }
  }
  if constexpr (kGrad) {
    const bool some    = some_s != 0;
    const float factor = some ? float(double(a.grad_loss[row]) * a.temperature) : 0.0f;
    const float l2s    = log2f(all.s);
    const auto q       = [&](float x) { return ex2((x - all.m) * c - l2s); };
    T* g               = a.grad + row * a.ldg;
    const bool same    = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
    for (int j = j0 + tid; j < j1 && warp < NW; j += NT) {
      const Vec v = rv.load(z, j);
      Vec o;
#pragma unroll
      for (int e = 0; e < VE; ++e)
        o.e[e] = FloatIo<T>::down(some ? q(FloatIo<T>::up(v.e[e])) * factor : 0.0f);
      rv.store(g, j, o, same);
    }
    __syncthreads();
    const int lo = rv.first(j0) > 0 ? rv.first(j0) : 0;
    const int hi = rv.first(j1) < a.vocab ? rv.first(j1) : a.vocab;
    for (int j = tid; j < k && some; j += NT + 32) {
      const int t = id[j];
      float w;
      if (t >= lo && t < hi && listed_weight(id, logp, k, j, &w)) g[t] = FloatIo<T>::down(factor * (q(zid[j]) - w));
    }
  }
}

// ---------------------------------------------------------------------------------------
// Gradient alone, from the lse of an earlier forward pass: every vector stands for itself. NT threads take the
// vectors, one more warp the list.
// ---------------------------------------------------------------------------------------
template <typename T, int NT, int NV>
__global__ void __launch_bounds__(NT + 32)
distill_grad_kernel(const Args<T> a, unsigned parts)
{
  constexpr int VE = Vec16Of<T>::value;
  extern __shared__ __align__(16) unsigned char grad_smem[];
  __shared__ int some_s;
  const int k = a.list.k;
  int* id     = reinterpret_cast<int*>(grad_smem);
  float* logp = reinterpret_cast<float*>(id + k);
  float* zid  = logp + k;
  grid_dep_sync();
  const int64_t row = int64_t(blockIdx.x) / parts;
  const int part    = int(int64_t(blockIdx.x) - row * parts);
  const T* z        = a.logits + row * a.ldl;
  const RowVecs<T> rv(z, a.vocab);
  const int j0  = part * (NT * NV);
  const int j1  = j0 + NT * NV < rv.n ? j0 + NT * NV : rv.n;
  const int tid = int(threadIdx.x);
  if (j0 >= j1) return;  // uniform over the CTA
  const int lo = rv.first(j0) > 0 ? rv.first(j0) : 0;
  const int hi = rv.first(j1) < a.vocab ? rv.first(j1) : a.vocab;
  // 1 / T in two fp32 pieces: rounded to one it would scale the row by its largest logit's share of the error
  // (-inf is taken as the lowest finite value: -inf times a zero piece would be NaN)
  const double inv = 1.0 / a.temperature;
  const float hi_t = float(inv), lo_t = float(inv - double(hi_t));
  const float lse = a.lse_in[row];
  const auto q    = [&](float x) {
    const float f = fmaxf(x, -FLT_MAX);
    return ex2(fmaf(f, lo_t, fmaf(f, hi_t, -lse)) * 1.4426950408889634f);
  };
  VecOf<T, VE> raw[NV];
  if (tid < NT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = j0 + i * NT + tid;
      if (j < j1) raw[i] = rv.load(z, j);
    }
  } else {
    for (int j = tid - NT; j < k; j += 32) {
      fetch_entry(a, row, j, &id[j], &logp[j]);
      zid[j] = id[j] >= lo && id[j] < hi ? FloatIo<T>::up(z[id[j]]) : 0.0f;
    }
    const bool some = weigh_list(id, logp, k, float(1.0 / a.temperature));
    if (tid == NT) some_s = some;
  }
  __syncthreads();
  const bool some    = some_s != 0;
  const float factor = some ? float(double(a.grad_loss[row]) * a.temperature) : 0.0f;
  T* g               = a.grad + row * a.ldg;
  const bool same    = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15u) == 0;
  if (tid < NT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = j0 + i * NT + tid;
      if (j < j1) {
        VecOf<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          o.e[e] = FloatIo<T>::down(some ? q(FloatIo<T>::up(raw[i].e[e])) * factor : 0.0f);
        rv.store(g, j, o, same);
      }
    }
  }
  __syncthreads();
  for (int j = tid; j < k && some; j += NT + 32) {
    const int t = id[j];
    float w;
    if (t >= lo && t < hi && listed_weight(id, logp, k, j, &w)) g[t] = FloatIo<T>::down(factor * (q(zid[j]) - w));
  }
}

// ---------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------
// Vectors of a row at the worst phase of the rows there are.
template <typename T>
inline int64_t most_vectors(const Args<T>& a)
{
  constexpr int VE    = Vec16Of<T>::value;
  const int align     = common_alignment({reinterpret_cast<uintptr_t>(a.logits),
                                          a.n_rows > 1 ? uintptr_t(a.ldl) * sizeof(T) : uintptr_t(0)});
  const int64_t phase = align >= 16 ? 0 : VE - 1;
  return ceil_div<int64_t>(phase + a.vocab, VE);
}

template <typename T>
inline Args<T> rows_from(const Args<T>& a, int64_t r0, int64_t n)
{
  Args<T> b = a;
  b.n_rows  = n;
  b.logits += r0 * a.ldl;
  if (b.grad) b.grad += r0 * a.ldg;
  if (b.loss) b.loss += r0;
  if (b.lse) b.lse += r0;
  if (b.lse_in) b.lse_in += r0;
  if (b.grad_loss) b.grad_loss += r0;
  b.list.ids     = static_cast<const char*>(a.list.ids) + r0 * a.list.ldi * (a.list.id64 ? 8 : 4);
  b.list.teacher = static_cast<const char*>(a.list.teacher) + r0 * a.list.ldt * (a.list.tdt == 0 ? 4 : 2);
  return b;
}

template <typename Kernel, typename T>
inline cudaError_t launch_clusters(Kernel kern, const Args<T>& a, int64_t ctas, int size, int threads, size_t smem,
                                   cudaStream_t stream)
{
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim            = dim3(unsigned(ctas));
  cfg.blockDim           = dim3(unsigned(threads));
  cfg.dynamicSmemBytes   = smem;
  cfg.stream             = stream;
  cudaLaunchAttribute at[2];
  at[0].id                                         = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x                           = unsigned(size);
  at[0].val.clusterDim.y                           = 1;
  at[0].val.clusterDim.z                           = 1;
  at[1].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs                                        = at;
  cfg.numAttrs = (tuning().dep_launch == 1 && ctas >= sm_count()) ? 2u : 1u;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

// Clusters of a persistent kernel that fit the device at once (asked once per kernel, cluster size, shared memory).
template <typename Kernel>
inline int64_t resident_clusters(Kernel kern, int size, int threads, size_t smem)
{
  struct Known {
    size_t smem;
    int n;
  };
  static std::mutex lock;
  static std::unordered_map<const void*, Known> known[64][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  std::lock_guard<std::mutex> g(lock);
  Known& have = known[dev][ilog2_floor(unsigned(size))][reinterpret_cast<const void*>(kern)];
  if (have.n == 0 || have.smem != smem) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(unsigned(size) * 1024u);
    cfg.blockDim           = dim3(unsigned(threads));
    cfg.dynamicSmemBytes   = smem;
    cudaLaunchAttribute at[1];
    at[0].id               = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(size);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs              = at;
    cfg.numAttrs           = 1;
    int n                  = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    have = {smem, n};
  }
  return have.n;
}

template <typename T, int NT>
inline cudaError_t launch_step(Args<T> a, int64_t most, int size, cudaStream_t stream)
{
  auto kern         = distill_step_kernel<T, NT>;
  const size_t smem = size_t(kStages) * NT * kStepNv * 16 + size_t(a.list.k) * 32;
  a.per_cta         = int(ceil_div<int64_t>(most, size));
  cudaError_t e     = ensure_dynamic_smem(kern, smem);
  if (e != cudaSuccess) return e;
  const int64_t fit      = resident_clusters(kern, size, NT, smem);
  const int64_t clusters = a.n_rows < fit ? a.n_rows : fit;
  return launch_clusters(kern, a, clusters * size, size, NT, smem, stream);
}

template <typename T, int NT, bool kGrad>
inline cudaError_t launch_stream(Args<T> a, int64_t most, int size, cudaStream_t stream)
{
  a.per_cta              = int(ceil_div<int64_t>(most, size));
  const size_t smem      = size_t(a.list.k) * 12;
  const int64_t max_rows = int64_t(0x7fffffff) / size;
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += max_rows) {
    const int64_t n     = a.n_rows - r0 < max_rows ? a.n_rows - r0 : max_rows;
    const cudaError_t e = launch_clusters(distill_stream_kernel<T, NT, kGrad>, rows_from(a, r0, n), n * size, size,
                                          NT + 32, smem, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Loss and gradient: a row is held by the CTAs of a cluster, NT x kStepNv vectors each; small vocabularies take small
// CTAs, and a row of more than 8 CTAs of 1024 threads is read twice.
template <typename T>
inline cudaError_t launch_loss_and_grad(const Args<T>& a, cudaStream_t stream)
{
  const int64_t most = most_vectors(a);
  // (beside 192 KB of buffers a CTA of 1024 threads has room for lists of 960 entries)
  if (a.list.k > 960) return launch_stream<T, 512, true>(a, most, 8, stream);
  if (most <= 128 * kStepNv) return launch_step<T, 128>(a, most, 1, stream);
  if (most <= 512 * kStepNv) return launch_step<T, 512>(a, most, 1, stream);
  for (int size = 1; size <= 8; size *= 2)
    if (most <= int64_t(1024) * kStepNv * size) return launch_step<T, 1024>(a, most, size, stream);
  return launch_stream<T, 512, true>(a, most, 8, stream);
}

// Loss: CTAs of 128 threads for short rows; rows are split over up to 8 CTAs while there are fewer than two per SM.
template <typename T>
inline cudaError_t launch_loss(const Args<T>& a, cudaStream_t stream)
{
  const int64_t most = most_vectors(a);
  if (most <= 128 * kStreamNv * 2) return launch_stream<T, 128, false>(a, most, 1, stream);
  int size = 1;
  while (size < 8 && a.n_rows * size < 2 * int64_t(sm_count()) && most >= int64_t(512) * kStreamNv * size)
    size *= 2;
  return launch_stream<T, 512, false>(a, most, size, stream);
}

template <typename T>
inline cudaError_t launch_grad_only(const Args<T>& a, cudaStream_t stream)
{
  constexpr int NT       = 256;
  constexpr int NV       = 4;
  const unsigned parts   = unsigned(ceil_div<int64_t>(most_vectors(a), NT * NV));
  const size_t smem      = size_t(a.list.k) * 12;
  const int64_t max_rows = int64_t(0x7fffffff) / parts;
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += max_rows) {
    const int64_t n = a.n_rows - r0 < max_rows ? a.n_rows - r0 : max_rows;
    (void)launch_dep(distill_grad_kernel<T, NT, NV>, dim3(unsigned(n * parts)), dim3(NT + 32), smem, stream,
                     rows_from(a, r0, n), parts);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace distill
}  // namespace detail
}  // namespace raft_b200
