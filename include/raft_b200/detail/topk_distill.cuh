// Distillation from a teacher's top logits.
//
// A row has student logits z over the vocabulary and a list of (token, teacher logit) pairs. With the temperature T
//     p = softmax(teacher / T) over the valid entries of the list         (token in [0, vocab))
//     q = softmax(z / T)       over the vocabulary
//     loss = T^2 * sum_k p_k (log p_k - log q[id_k]),     lse = log sum_v exp(z_v / T)
//     d loss / d z_v = T (q_v - sum of p_k with id_k = v)
// A p_k that fp32 holds as 0 (an entry far below the list's largest) adds nothing, where q is 0 too: not 0 * inf.
// A row without a valid entry (all tokens -1: prompt or padding positions) has loss 0 and gradient 0.
//
// The pass over the logits is what costs: V elements per row are read once, and written once where the gradient is
// wanted. For the gradient a row is spread over the CTAs of a cluster, which keep it in shared memory between the two
// uses, so that no second read is needed; the CTAs exchange (maximum, sum) pairs through distributed shared memory.
// Sums and statistics are fp32, relative to the maximum; the loss, a sum of k terms, is fp64.
#pragma once

#include "launch.cuh"
#include "row_normalize_staged.cuh"
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
  RingCtl ctl;  // bounded waits
  int late_warp;  // test hook (-1: none): this warp of the first CTA is told that row ctl.skip_tile did not arrive in time
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

// 16 bytes to the same place of CTA `rank`, counted by the barrier at the same place there: the data has arrived when
// the barrier's phase completes. No fence is involved, so global stores under way are not waited for.
B2R_DI void cluster_send(float4* p, uint64_t* bar, unsigned rank, float4 v)
{
  unsigned to, at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(at)
               : "memory");
}

B2R_DI void cluster_send(double* p, uint64_t* bar, unsigned rank, double v)
{
  unsigned to, at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to),
               "l"(__double_as_longlong(v)), "r"(at)
               : "memory");
}

// A part of a row as 16-byte vectors of its memory. Vector j of a row holds elements [j * VE - phase, (j + 1) * VE -
// phase), where `phase` elements lie between the 16-byte boundary at or before the row's first element and that
// element. Only whole vectors are moved as vectors: the first vector of a row and its last may not be, their elements
// are moved one by one, so nothing outside the row is touched.
template <typename T>
struct RowPart {
  static constexpr int VE = Vec16Of<T>::value;
  const T* at;     // where element 0 of the part's first vector is, or would be
  int first;       // its token (negative: before the row)
  int n;           // vectors of the part
  int lo, hi;      // those that are whole: [lo, hi)
  int token0, token1;  // tokens of the part

  // vectors [j0, j0 + most) of the row
  B2R_DI RowPart(const T* row, int vocab, int j0, int most) : RowPart(row, phase_of(row), vocab, j0, most) {}
  B2R_DI static int phase_of(const T* row) { return int(uintptr_t(row) & 15u) / int(sizeof(T)); }
  B2R_DI RowPart(const T* row, int phase, int vocab, int j0, int most)
  {
    const int end   = phase + vocab;  // behind the row, in elements from the boundary
    const int all   = (end + VE - 1) / VE;
    n               = all - j0 < most ? (all > j0 ? all - j0 : 0) : most;
    first           = j0 * VE - phase;
    at              = row + first;
    lo              = first < 0 && n > 0 ? 1 : 0;
    hi              = n - (n > 0 && j0 + n == all && end % VE != 0 ? 1 : 0);
    token0          = first > 0 ? first : 0;
    token1          = first + n * VE < vocab ? first + n * VE : vocab;
  }
  B2R_DI bool whole(int i) const { return i >= lo && i < hi; }
  B2R_DI bool edges() const { return lo != 0 || hi < n; }

  B2R_DI Words4 load_whole(int i) const
  {
    Words4 r;
    // not the non-coherent path: the gradient may be written over the logits
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                 : "l"(at + i * VE)
                 : "memory");
    return r;
  }
  // a vector that may reach over an end of the row: -inf there
  B2R_DI Words4 load_edge(int i) const
  {
    Words4 r;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int t = first + i * VE + e;
      put_bits<T>(r, e, t >= token0 && t < token1 ? at[i * VE + e] : FloatIo<T>::down(-INFINITY));
    }
    return r;
  }
  B2R_DI Words4 load(int i) const { return whole(i) ? load_whole(i) : load_edge(i); }
  // element by element, as much of it as belongs to the part; `dst` where `at` is in the output's row
  B2R_DI void store_edge(T* dst, int i, const Words4& v) const
  {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int t = first + i * VE + e;
      if (t >= token0 && t < token1) dst[i * VE + e] = get_bits<T>(v, e);
    }
  }
  // `same`: the output's row has the same phase
  B2R_DI void store(T* dst, int i, const Words4& v, bool same) const
  {
    if (same && whole(i))
      *reinterpret_cast<Words4*>(dst + i * VE) = v;
    else
      store_edge(dst, i, v);
  }
};
template <typename T>
B2R_DI Words4 minus_inf()
{
  Words4 r;
#pragma unroll
  for (int q = 0; q < Vec16Of<T>::value / 2; ++q)
    down_pair<T>(r, q, make_float2(-INFINITY, -INFINITY));
  return r;
}
B2R_DI bool same_phase(const void* a, const void* b)
{
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15u) == 0;
}

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

// NaN operands lose, as in fmaxf
B2R_DI float warp_max(float v)
{
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
B2R_DI float max3(float a, float b, float c)
{
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// NaN if either is
B2R_DI float max_nan(float a, float b)
{
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
B2R_DI float min_nan(float a, float b)
{
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two fp32 values handled by one instruction.
using Pair = unsigned long long;
B2R_DI Pair pair(float a, float b)
{
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
B2R_DI float2 split(Pair p)
{
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
B2R_DI Pair add2(Pair a, Pair b)
{
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
B2R_DI Pair mul2(Pair a, Pair b)
{
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
B2R_DI Pair fma2(Pair a, Pair b, Pair c)
{
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// 2^x of both
B2R_DI Pair ex2_2(Pair x)
{
  const float2 v = split(x);
  return pair(ex2(v.x), ex2(v.y));
}

template <typename T>
B2R_DI Pair up2(const Words4& v, int q)
{
  const float2 f = up_pair<T>(v, q);
  return pair(f.x, f.y);
}
template <typename T>
B2R_DI void down2(Words4& v, int q, Pair p)
{
  down_pair<T>(v, q, split(p));
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

// Entry j of a row's list, as it lies in memory: loads under way do not stop the warp until a value is looked at, and a
// conversion is such a look.
struct Entry {
  unsigned lo, hi;  // token (hi: of int64 tokens)
  unsigned y;       // bits of the teacher's logit

  template <typename T>
  B2R_DI void ask(const Args<T>& a, int64_t row, int j)
  {
    if (a.list.id64) {
      const uint2 t = *reinterpret_cast<const uint2*>(static_cast<const long long*>(a.list.ids) + row * a.list.ldi + j);
      lo            = t.x;
      hi            = t.y;
    } else {
      lo = static_cast<const unsigned*>(a.list.ids)[row * a.list.ldi + j];
    }
    if (a.list.tdt == 0)
      y = static_cast<const unsigned*>(a.list.teacher)[row * a.list.ldt + j];
    else
      y = static_cast<const uint16_t*>(a.list.teacher)[row * a.list.ldt + j];
  }
  template <typename T>
  B2R_DI int id(const Args<T>& a) const  // -1: not valid
  {
    const bool ok = (!a.list.id64 || hi == 0u) && lo < unsigned(a.vocab);
    return ok ? int(lo) : -1;
  }
  template <typename T>
  B2R_DI float logit(const Args<T>& a) const
  {
    if (a.list.tdt == 0) return __uint_as_float(y);
    if (a.list.tdt == 7) return __uint_as_float(y << 16);  // B2R_BF16
    const __half_raw h{static_cast<unsigned short>(y)};
    return __half2float(__half(h));
  }
};

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
// walk the rows. Rows come into a ring of kStages shared-memory buffers by bulk copies; the workers go over a row twice
// there. The first time each takes (m, s) of its elements; the CTA's (m, s) goes to every CTA of the cluster as a record
// that a shared-memory barrier counts. The second time they write the gradient over the row, and a bulk copy takes it
// to memory. Between the two lies the first pass over the NEXT row, so that nobody waits for the records.
//
// Two exponentials per element: 8 elements per clock and SM at the MUFU unit's 16, 4100 clocks of a row's 64 KB part,
// against 5100 that its 128 KB of traffic take. 4096 x 131072 bf16 takes 513 us (4.2 TB/s; clusters of four fit on 132
// of the 148 SMs, with 19 warps each; neither the exponential unit, 51 %, nor the memory, 41 %, is the limit). Keeping
// the first pass's exponentials instead needs 64 registers of every worker for them; ptxas then spills (512 workers of 64
// elements: 96 registers, 815 us for 4096 rows of 131072 bf16; 256 of 128: 168 registers, 1195 us). Forms before that:
// workers that copied their own vectors in and out, 750 us (5000 of 12000 clocks per row in the copies); cluster barriers
// for the exchange, which wait for the gradient's stores, 1350 us.
//
// Three warps work beside the workers, so that no chain of loads is on the workers' path:
//   the sender   joins the CTA's (m, s), sends the record, and in the first CTA writes the loss;
//   the mover    issues the copies, and waits until a row's gradient has been read before the next row comes in;
//   the lister   prepares the list of the row after the next: weights, the student's logits of the listed tokens, and
//                the sums A = sum p (log p - z / T), P = sum p over the tokens this CTA holds, of which the loss is
//                T^2 (A + P lse). (The listed elements of the gradient are written by the warp that holds them.)
//
// Every wait is bounded. Whoever gives up sets `gave_up`, by which the CTA reports at its end. A warp that did not see
// its row come in leaves NaN in the row's record and marks the buffer as missed; the mover then writes NaN over the
// CTA's part of that row and asks for no further ones.
//
// kEven: all rows have the phase of the first, so that the geometry is worked out once.
// ---------------------------------------------------------------------------------------
constexpr int kStages = 3;  // vectors of the row in its second pass, of the next in its first, of the one after under way
constexpr int kStepNv = 8;  // vectors of a worker, in chunks of four

template <typename T, int NT, bool kEven>
__global__ void __launch_bounds__(NT + 96, NT == 256 ? 2 : 1)
distill_step_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  constexpr int NV = kStepNv;
  constexpr int NW = NT / 32;
  constexpr int CV = 4;            // vectors of a chunk
  constexpr int CP = CV * VE / 2;  // pairs of a chunk
  using Vec        = Words4;
  extern __shared__ __align__(128) unsigned char step_smem[];
  // Records by row & 3: a CTA that is ahead may send the row after the next while another still reads the row before.
  __shared__ __align__(16) float4 record[4][8];   // by CTA rank: m, s, A (fp64)
  __shared__ __align__(8) double record_p[4][8];  // P
  __shared__ __align__(8) uint64_t arrived[4];
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ float2 warp_part[NW];
  __shared__ double list_sums[3][2];  // A, P
  __shared__ float factor_s[3];       // weight of the row's gradient, 0 for a row without a list
  __shared__ int some_s[3];
  __shared__ int twice_s[3];  // a token of this CTA's is named twice
  __shared__ int gave_up;
  __shared__ int missed[kStages];  // somebody did not see the copy into this buffer arrive
  Vec* stages         = reinterpret_cast<Vec*>(step_smem);                   // [kStages][NT * NV]
  const int k         = a.list.k;
  int* ids            = reinterpret_cast<int*>(stages + kStages * NT * NV);  // [3][k]
  float* logps        = reinterpret_cast<float*>(ids + 3 * k);               // [3][k]
  float* zids         = logps + 3 * k;                                       // [3][k]
  unsigned* seen      = reinterpret_cast<unsigned*>(zids + 3 * k);           // a bit per element of the part
  const unsigned rank = cluster_rank();
  const unsigned size = cluster_size();
  const int tid       = int(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i)
      mbar_init(&arrived[i], 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      missed[i] = 0;
    }
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int64_t step  = int64_t(gridDim.x) / size;
  const int64_t first = int64_t(blockIdx.x) / size;
  const float c       = float(1.4426950408889634 / a.temperature);
  const int j0        = int(rank) * a.per_cta;
  const auto part_of  = [&](int64_t row) {
    const T* z = a.logits + row * a.ldl;
    return RowPart<T>(z, RowPart<T>::phase_of(kEven ? a.logits : z), a.vocab, j0, a.per_cta);
  };
  // Places behind the end of a part hold -inf, which adds nothing: no vector has to be asked about when it is used.
  // Nobody writes there again, but for rows of different phases, whose parts differ by a vector.
  {
    const RowPart<T> part = part_of(0);
    for (int i = tid; i < NT * NV; i += NT + 96)
      if (i >= part.n) stages[i] = stages[NT * NV + i] = stages[2 * NT * NV + i] = minus_inf<T>();
  }
  for (int i = tid; i < NT * NV * VE / 32; i += NT + 96)
    seen[i] = 0;
  fence_proxy_async();
  __syncthreads();
  cluster_arrive();  // every CTA of the cluster has started, its barriers are set up
  grid_dep_sync();

  const int late_row = blockIdx.x == 0 && warp == a.late_warp ? a.ctl.skip_tile : -1;
  bool there = true;  // everything that this warp has waited for so far has arrived
  // Whether row number n of this cluster, on its way into buffer `stage`, has arrived. The copy may still land after a
  // wait that ran out, over whatever the buffer holds then: `missed` keeps the buffer from becoming a gradient.
  auto landed = [&](int n, int stage, unsigned phase) {
    const bool late = n == late_row;
    if (late) *static_cast<volatile int*>(&gave_up) = 1;
    const bool here = there && !late && mbar_wait_bounded(&full[stage], phase, &gave_up, a.ctl.limit_ns);
    if (!here) *static_cast<volatile int*>(&missed[stage]) = 1;
    return here;
  };

  // ---- mover
  // row's vectors on their way into buffer `stage` (all lanes of the warp come here)
  auto request = [&](int64_t row, int stage) {
    if (row >= a.n_rows) return;
    const RowPart<T> part = part_of(row);
    Vec* to               = stages + stage * (NT * NV);
    if (lane == 0 && part.lo != 0) to[0] = part.load_edge(0);
    if (lane == 1 && part.hi < part.n && (part.n > 1 || part.lo == 0)) to[part.n - 1] = part.load_edge(part.n - 1);
    if (!kEven && lane == 2 && part.n < NT * NV) to[part.n] = minus_inf<T>();
    __syncwarp();  // these are there, too, for whoever has seen the barrier
    if (lane == 0) {
      const int whole = part.hi > part.lo ? part.hi - part.lo : 0;
      mbar_expect_tx(&full[stage], unsigned(whole) * 16u);
      for (int i = 0; i < whole; i += 1024) {
        const int n = whole - i < 1024 ? whole - i : 1024;
        bulk_load(to + part.lo + i, part.at + (part.lo + i) * VE, unsigned(n) * 16u, &full[stage]);
      }
    }
  };
  // the gradient of a row from its buffer to memory, as far as that goes in whole vectors
  auto write_back = [&](int64_t row, int stage) {
    const RowPart<T> part = part_of(row);
    T* g                  = a.grad + row * a.ldg;
    if (lane == 0 && part.hi > part.lo && same_phase(g, a.logits + row * a.ldl))
      bulk_store(g + part.first + part.lo * VE, stages + stage * (NT * NV) + part.lo, unsigned(part.hi - part.lo) * 16u);
  };
  // NaN over what has become of a row that somebody missed
  auto take_back = [&](int64_t row) {
    bulk_store_wait_all();
    __syncwarp();
    const RowPart<T> part = part_of(row);
    T* g                  = a.grad + row * a.ldg;
    for (int64_t t = part.token0 + lane; t < part.token1; t += 32)
      g[t] = FloatIo<T>::down(NAN);
  };

  // ---- sender
  // the record of a row whose parts the workers have left in warp_part (all lanes); n: the row's number here
  auto send = [&](int n, int buf) {
    const float2 v = lane < NW ? warp_part[lane] : make_float2(-INFINITY, 0.0f);
    const ExpSum w = warp_join({v.x, v.y}, c);
    const long long bits = __double_as_longlong(list_sums[buf][0]);
    const float4 rec = make_float4(w.m, w.s, __int_as_float(int(bits)), __int_as_float(int(bits >> 32)));
    const int at     = n & 3;
    // test hook: this record is never sent
    const bool skip = blockIdx.x == 0 && n == a.ctl.skip_tile && a.late_warp < 0;
    if (size == 1) {
      if (lane == 0 && !skip) {
        record[at][0]   = rec;
        record_p[at][0] = list_sums[buf][1];
        mbar_arrive(&arrived[at]);
      }
    } else {
      if (lane == 0) mbar_expect_tx(&arrived[at], size * 24u);
      if (lane < int(size) && !skip) {
        cluster_send(&record[at][rank], &arrived[at], unsigned(lane), rec);
        cluster_send(&record_p[at][rank], &arrived[at], unsigned(lane), list_sums[buf][1]);
      }
    }
  };

  // ---- lister
  const double inverse = 1.0 / a.temperature;
  // The first entries of a row's list and its weight are asked for a turn before they are used, and worked on in
  // registers; those of long lists behind them go through shared memory.
  constexpr int kAhead = 4;
  Entry ahead[kAhead];
  float ahead_weight = 0.0f;
  auto ask           = [&](int64_t row) {
    if (row >= a.n_rows) return;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u * 32 + lane < k) ahead[u].ask(a, row, u * 32 + lane);
    ahead_weight = a.grad_loss[row];
  };
  auto prepare = [&](int64_t row, int n, int buf, int stage, unsigned phase) {
    if (row >= a.n_rows) return;
    const RowPart<T> part = part_of(row);
    int* id               = ids + buf * k;
    float* logp           = logps + buf * k;
    float* zid            = zids + buf * k;
    int near_id[kAhead];
    float near_y[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      near_id[u] = u * 32 + lane < k ? ahead[u].id(a) : -1;
      near_y[u]  = ahead[u].logit(a);
    }
    const float weight = ahead_weight;
    ask(row + step);
    for (int j = kAhead * 32 + lane; j < k; j += 32) {
      Entry entry;
      entry.ask(a, row, j);
      id[j]   = entry.id(a);
      logp[j] = entry.logit(a);
    }
    // f(place, token, logit or log weight) for every valid entry; the value may be changed
    const auto each = [&](auto f) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (near_id[u] >= 0) f(u * 32 + lane, near_id[u], near_y[u]);
      for (int j = kAhead * 32 + lane; j < k; j += 32)
        if (id[j] >= 0) f(j, id[j], logp[j]);
    };
    const float inv_t = float(inverse);
    float m           = -INFINITY;
    bool nan          = false;
    each([&](int, int, float& y) {
      m   = fmaxf(m, y);
      nan = nan || y != y;
    });
    m               = warp_max(m);
    nan             = __any_sync(kFull, nan);
    const bool some = m > -INFINITY || nan;
    float total     = 0.0f;
    each([&](int, int, float& y) { total += some ? expf((y - m) * inv_t) : 0.0f; });
    const float ls = logf(warp_sum(total));
    // the row itself, for the student's logits of the listed tokens
    const bool here = landed(n, stage, phase);
    const T* held   = reinterpret_cast<const T*>(stages + stage * (NT * NV)) - part.first;  // held[t]: token t
    double sum = 0.0, share = 0.0;
    bool twice = false;
    each([&](int j, int t, float& y) {
      const float lp = some ? (y - m) * inv_t - ls : -INFINITY;
      logp[j]        = lp;
      if (t >= part.token0 && t < part.token1 && some && here) {
        const unsigned at = unsigned(t - part.first), bit = 1u << (at & 31u);
        twice          = twice || (atomicOr(&seen[at >> 5], bit) & bit) != 0u;
        const float zt = FloatIo<T>::up(held[t]);
        const double w = double(expf(lp));
        zid[j]         = zt;
        sum += w == 0.0 ? 0.0 : w * (double(lp) - double(zt) * inverse);
        share += w;
      }
    });
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u * 32 + lane < k) id[u * 32 + lane] = near_id[u];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(kFull, sum, o);
      share += __shfl_xor_sync(kFull, share, o);
    }
    twice = __any_sync(kFull, twice);
    __syncwarp();  // the bits are cleared when all lanes have asked for theirs, and asked for again when they are clear
    each([&](int, int t, float&) {
      if (t >= part.token0 && t < part.token1) seen[unsigned(t - part.first) >> 5] = 0;
    });
    __syncwarp();
    if (lane == 0) {
      twice_s[buf]      = twice;
      list_sums[buf][0] = here ? sum : double(NAN);
      list_sums[buf][1] = share;
      some_s[buf]       = some;
      factor_s[buf]     = some ? float(double(weight) * a.temperature) : 0.0f;
    }
  };

  // ---- workers
  // (m, s) of the warp's elements of row number n here, which lies in buffer `stage`
  auto first_pass = [&](int64_t row, int n, int stage, unsigned phase) {
    const int n_vec = part_of(row).n;
    there           = landed(n, stage, phase);
    const Vec* mine = stages + stage * (NT * NV) + tid;
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int i0 = 0; i0 < NV; i0 += CV) {
      if (i0 * NT + warp * 32 >= n_vec) break;
      Pair e[CP];
      float top = m;
#pragma unroll
      for (int i = 0; i < CV; ++i) {
        const Vec v = mine[(i0 + i) * NT];
#pragma unroll
        for (int q = 0; q < VE / 2; ++q) {
          e[i * VE / 2 + q] = up2<T>(v, q);
          const float2 f    = split(e[i * VE / 2 + q]);
          top               = max3(top, f.x, f.y);
        }
      }
      if (top > m) {
        s = m == -INFINITY ? s : s * ex2((m - top) * c);
        m = top;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      const Pair sub = pair(-base, -base), mul = pair(c, c);
      Pair sum0 = pair(s, 0.0f), sum1 = pair(0.0f, 0.0f);
#pragma unroll
      for (int q = 0; q < CP; q += 2) {
        sum0 = add2(sum0, ex2_2(mul2(add2(e[q], sub), mul)));
        sum1 = add2(sum1, ex2_2(mul2(add2(e[q + 1], sub), mul)));
      }
      const float2 s2 = split(add2(sum0, sum1));
      s               = s2.x + s2.y;
    }
    const ExpSum w = warp_join({m, there ? s : NAN}, c);
    if (lane == 0) warp_part[warp] = make_float2(w.m, w.s);
  };
  // the gradient of the row in buffer `stage`, written over it (vectors that are not whole, or whose row in memory has
  // another phase: straight to memory, an element at a time)
  auto second_pass = [&](int64_t row, int n, int buf, int stage, unsigned phase) {
    there            = there && mbar_wait_bounded(&arrived[n & 3], phase, &gave_up, a.ctl.limit_ns);
    const float4 r   = lane < int(size) ? record[n & 3][lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    ExpSum all       = warp_join({r.x, r.y}, c);
    if (!there) all.s = NAN;
    const bool some  = some_s[buf] != 0;
    const float fact = factor_s[buf];
    const float l2s  = log2f(all.s);
    const Pair sub = pair(-all.m, -all.m), mul = pair(c, c), off = pair(-l2s, -l2s), fact2 = pair(fact, fact);
    const RowPart<T> part = part_of(row);
    Vec* mine             = stages + stage * (NT * NV) + tid;
    T* to                 = a.grad + row * a.ldg + part.first;
    const bool same       = same_phase(to, part.at);
    const bool plain      = same && !part.edges();  // everything is written by the bulk copy
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * NT + warp * 32 < part.n) {
        const Vec v = mine[i * NT];
        Vec o;
#pragma unroll
        for (int q = 0; q < VE / 2; ++q)
          down2<T>(o, q, mul2(ex2_2(fma2(add2(up2<T>(v, q), sub), mul, off)), fact2));
        if (!some) o = Vec{};
        if (i * NT + tid < part.n) mine[i * NT] = o;
      }
    }
    if (!plain) {
#pragma unroll 1
      for (int j = tid; j < part.n; j += NT)
        if (!(same && part.whole(j))) part.store_edge(to, j, mine[j - tid]);
    }
    // the listed elements of the warp's vectors: q - sum of the token's weights
    __syncwarp();
    if (some) {
      const int* id     = ids + buf * k;
      const float* logp = logps + buf * k;
      const float* zid  = zids + buf * k;
      const bool twice  = twice_s[buf] != 0;
      for (int l0 = 0; l0 < k; l0 += 32) {
        const int t0  = l0 + lane < k ? id[l0 + lane] : -1;
        const bool my = t0 >= part.token0 && t0 < part.token1 && (unsigned(t0 - part.first) / VE) % NT / 32 == unsigned(warp);
        const auto put = [&](int t, float zt, float w) {
          const T v    = FloatIo<T>::down(fact * (ex2((zt - all.m) * c - l2s) - w));
          const int at = t - part.first;
          if (same && part.whole(at / VE))
            reinterpret_cast<T*>(stages + stage * (NT * NV))[at] = v;
          else
            to[at] = v;
        };
        if (!twice) {
          if (my) put(t0, zid[l0 + lane], expf(logp[l0 + lane]));
          continue;
        }
        for (unsigned left = __ballot_sync(kFull, my); left != 0u; left &= left - 1u) {
          const int j = l0 + __ffs(int(left)) - 1;
          const int t = id[j];
          float w     = 0.0f;
          int before  = 0;  // entries of the token ahead of this one: the first speaks for all
          for (int i = lane; i < k; i += 32) {
            if (id[i] == t) {
              w += expf(logp[i]);
              before += i < j;
            }
          }
          w = warp_sum(w);
          if (!__any_sync(kFull, before != 0) && lane == 0) put(t, zid[j], w);
        }
      }
    }
    fence_proxy_async();
  };

  // workers and sender
  const auto handover = [] { asm volatile("bar.sync 1, %0;" ::"n"(NT + 32) : "memory"); };

  // Row number n of this cluster lies in buffer n % 3, as does its list; its records at n & 3.
  if (warp == NW + 2) {
    for (int n = 0; n < kStages; ++n)
      request(first + n * step, n);
  }
  __syncthreads();
  if (warp == NW + 1) ask(first);
  if (warp == NW + 1) prepare(first, 0, 0, 0, 0);
  if (warp == NW + 1) prepare(first + step, 1, 1, 1, 0);
  if (warp < NW) first_pass(first, 0, 0, 0);
  cluster_wait();
  __syncthreads();
  if (warp == NW) send(0, 0);

  int cur        = 0;   // n % 3, and the parity of its round
  unsigned round = 0;
  int n          = 0;
  for (int64_t row = first; row < a.n_rows; row += step, ++n) {
    const int nxt         = cur + 1 == kStages ? 0 : cur + 1;
    const unsigned nround = nxt == 0 ? round ^ 1u : round;
    const int nn          = nxt + 1 == kStages ? 0 : nxt + 1;
    const unsigned phase  = unsigned(n >> 2) & 1u;  // of the records
    bool listed = false;
    if (warp < NW) {
      if (row + step < a.n_rows) first_pass(row + step, n + 1, nxt, nround);
      handover();
      second_pass(row, n, cur, cur, phase);
    } else if (warp == NW) {
      handover();
      if (row + step < a.n_rows && there) send(n + 1, nxt);
      listed = some_s[cur] != 0;
    } else if (warp == NW + 1 && there) {
      // (the list of the row after the next goes where the row before had its)
      prepare(row + 2 * step, n + 2, nn, nn, nn == 0 || nxt == 0 ? round ^ 1u : round);
    }
    __syncthreads();
    if (warp == NW + 2) {
      write_back(row, cur);
      bulk_store_wait_read();  // (by the lane that stores)
      __syncwarp();
      // (after a give-up nothing says that the buffer's last copy has landed)
      // (both flags may be set meanwhile: the warp decides as a whole)
      if (!__any_sync(kFull, *static_cast<volatile int*>(&gave_up) != 0))
        request(row + 3 * step, cur);
      else if (__any_sync(kFull, *static_cast<volatile int*>(&missed[cur]) != 0))
        take_back(row);
    } else if (warp == NW) {
      there = there && mbar_wait_bounded(&arrived[n & 3], phase, &gave_up, a.ctl.limit_ns);
      if (rank == 0) {
        const float4 r   = lane < int(size) ? record[n & 3][lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        const double p   = lane < int(size) ? record_p[n & 3][lane] : 0.0;
        const ExpSum all = warp_join({r.x, r.y}, c);
        const double sum = warp_sum(__longlong_as_double((long long)(unsigned(__float_as_int(r.z))) |
                                                         ((long long)(__float_as_int(r.w)) << 32)));
        const double wgt = warp_sum(p);
        const double lse = there ? double(all.m) * inverse + double(logf(all.s)) : double(NAN);
        if (lane == 0) {
          if (a.loss != nullptr) a.loss[row] = listed ? float((sum + wgt * lse) * a.temperature * a.temperature) : 0.0f;
          if (a.lse != nullptr) a.lse[row] = float(lse);
        }
      }
    }
    cur   = nxt;
    round = nround;
  }
  if (warp == NW + 2) {
    bulk_store_wait_all();
    if (*static_cast<volatile int*>(&gave_up) != 0 && lane == 0) {
      // copies still on their way in must have landed before the CTA leaves: the last of each buffer, if any
      for (int i = 0; i < kStages; ++i)
        (void)mbar_drain_bounded(&full[i], i < cur ? round : round ^ 1u, a.ctl.limit_ns);
    }
  }
  __syncthreads();
  if (tid == 0 && gave_up != 0) ring_report_timeout(a.ctl);  // whoever it was
  if (size > 1) {  // nobody sends to a CTA that has left
    cluster_arrive();
    cluster_wait();
  }
}

// ---------------------------------------------------------------------------------------
// Gradients whose rows or lists do not fit the shared memory of a cluster (kGrad), and the loss alone: NT threads stream
// their CTA's part of the row through shared memory (every thread its own vectors, kStreamDepth - 1 chunks of kStreamNv
// vectors under way), and one more warp of rank 0's CTA takes the list. With kGrad every part is read a second time.
// Chunks are short so that four CTAs fit an SM and one's beginning lies behind the others' chunks: 2048 x 131072 bf16 takes 113 us (4.8 TB/s),
// 141 with chunks of eight vectors and two CTAs per SM, 130 with four vectors and a fourth stage.
// ---------------------------------------------------------------------------------------
constexpr int kStreamNv    = 4;
constexpr int kStreamDepth = 3;

template <typename T, int NT, bool kGrad>
__global__ void __launch_bounds__(NT + 32)
distill_stream_kernel(const Args<T> a)
{
  constexpr int VE = Vec16Of<T>::value;
  constexpr int NV = kStreamNv;
  constexpr int NW = NT / 32;
  using Vec        = Words4;
  extern __shared__ __align__(16) unsigned char stream_smem[];
  __shared__ float2 parts[8 * NW];
  __shared__ int some_s;
  const unsigned rank = cluster_rank();
  const unsigned size = cluster_size();
  const int tid       = int(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31;
  const int k   = a.list.k;
  Vec* ring     = reinterpret_cast<Vec*>(stream_smem);                 // [kStreamDepth][NT * NV]
  int* id       = reinterpret_cast<int*>(ring + kStreamDepth * NT * NV);  // [k]
  float* logp   = reinterpret_cast<float*>(id + k);     // [k]
  float* zid    = logp + k;                             // [k] student logits of the listed tokens
  cluster_arrive();
  grid_dep_sync();
  const int64_t row = int64_t(blockIdx.x) / size;
  const T* z        = a.logits + row * a.ldl;
  const RowPart<T> part(z, a.vocab, int(rank) * a.per_cta, a.per_cta);
  const float c = float(1.4426950408889634 / a.temperature);
  if (warp == NW) {  // the list
    if (kGrad || rank == 0) {
      for (int j = lane; j < k; j += 32) {
        Entry entry;
        entry.ask(a, row, j);
        const int at = entry.id(a);
        id[j]        = at;
        zid[j]       = at >= 0 ? FloatIo<T>::up(z[at]) : 0.0f;
        logp[j]      = entry.logit(a);
      }
      const bool some = weigh_list(id, logp, k, float(1.0 / a.temperature));
      if (lane == 0) some_s = some;
    }
    cluster_wait();
  } else {
    float m = -INFINITY, s = 0.0f;  // as ExpSum
    auto request = [&](int j, int stage) {  // vectors [j, j + NV * NT) of the part
      Vec* to       = ring + stage * (NT * NV) + tid;
      const T* from = part.at + (j + tid) * VE;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (part.whole(j + i * NT + tid)) copy_async16(to + i * NT, from + i * (NT * VE));
      if (part.edges() || j + NV * NT > part.n) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int q = j + i * NT + tid;
          if (!part.whole(q)) to[i * NT] = q < part.n ? part.load_edge(q) : minus_inf<T>();
        }
      }
      copy_commit();
    };
    const Pair mul = pair(c, c);
    auto use = [&](const Vec* slot, int j) {
      Pair e[NV * VE / 2];
      float top = m;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Vec v = slot[i * NT + tid];  // -inf behind the end of the part
#pragma unroll
        for (int q = 0; q < VE / 2; ++q) {
          e[i * VE / 2 + q] = up2<T>(v, q);
          const float2 f    = split(e[i * VE / 2 + q]);
          top               = max3(top, f.x, f.y);
        }
      }
      if (top > m) {
        s = m == -INFINITY ? s : s * ex2((m - top) * c);
        m = top;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      const Pair sub   = pair(-base, -base);
      Pair sum0 = pair(s, 0.0f), sum1 = pair(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (j + i * NT + warp * 32 < part.n) {
#pragma unroll
          for (int q = i * VE / 2; q < (i + 1) * VE / 2; q += 2) {
            sum0 = add2(sum0, ex2_2(mul2(add2(e[q], sub), mul)));
            sum1 = add2(sum1, ex2_2(mul2(add2(e[q + 1], sub), mul)));
          }
        }
      }
      const float2 s2 = split(add2(sum0, sum1));
      s               = s2.x + s2.y;
    };
    constexpr int kChunk = NV * NT;
#pragma unroll
    for (int d = 0; d < kStreamDepth - 1; ++d)
      request(d * kChunk, d);
    int stage = 0;
    for (int j = 0; j < part.n; j += kChunk) {
      copy_wait<kStreamDepth - 2>();
      use(ring + stage * kChunk, j);
      request(j + (kStreamDepth - 1) * kChunk, stage == 0 ? kStreamDepth - 1 : stage - 1);
      stage = stage + 1 == kStreamDepth ? 0 : stage + 1;
    }
    copy_wait<0>();
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
      const double w = double(expf(logp[j]));
      if (id[j] >= 0 && w != 0.0) sum += w * (double(logp[j]) - (double(zid[j]) / a.temperature - lse));
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
    const bool same    = same_phase(g, z);
    for (int j = tid; j < part.n && warp < NW; j += NT) {
      const Vec v = part.load(j);
      Vec o;
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        const float2 f = up_pair<T>(v, e);
        down_pair<T>(o, e, some ? make_float2(q(f.x) * factor, q(f.y) * factor) : make_float2(0.0f, 0.0f));
      }
      part.store(g + part.first, j, o, same);
    }
    __syncthreads();
    for (int j = tid; j < k && some; j += NT + 32) {
      const int t = id[j];
      float w;
      if (t >= part.token0 && t < part.token1 && listed_weight(id, logp, k, j, &w))
        g[t] = FloatIo<T>::down(factor * (q(zid[j]) - w));
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
  const T* z        = a.logits + row * a.ldl;
  const RowPart<T> part(z, a.vocab, int(int64_t(blockIdx.x) - row * parts) * (NT * NV), NT * NV);
  const int tid = int(threadIdx.x);
  if (part.n <= 0) return;  // uniform over the CTA
  // 1 / T in two fp32 pieces: rounded to one it would scale the row by its largest logit's share of the error
  // (-inf is taken as the lowest finite value: -inf times a zero piece would be NaN; a NaN stays one)
  const double inv = 1.0 / a.temperature;
  const float hi_t = float(inv), lo_t = float(inv - double(hi_t));
  // (a row of -inf alone has no probabilities)
  const float lse = a.lse_in[row] == -INFINITY ? NAN : a.lse_in[row];
  // The fp32 lse is off by up to |lse| 2^-24, which at low temperatures is more than 1: a probability never is.
  const auto q = [&](float x) {
    const float f = max_nan(x, -FLT_MAX);
    const float d = min_nan(fmaf(f, lo_t, fmaf(f, hi_t, -lse)), 0.0f);
    return ex2(fmaf(f, 0.0f, d * 1.4426950408889634f));  // (NaN for +inf)
  };
  Words4 raw[NV];
  if (tid < NT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * NT + tid;
      if (j < part.n) raw[i] = part.load(j);
    }
  } else {
    for (int j = tid - NT; j < k; j += 32) {
      Entry entry;
      entry.ask(a, row, j);
      const int at = entry.id(a);
      id[j]        = at;
      zid[j]       = at >= part.token0 && at < part.token1 ? FloatIo<T>::up(z[at]) : 0.0f;
      logp[j]      = entry.logit(a);
    }
    const bool some = weigh_list(id, logp, k, float(1.0 / a.temperature));
    if (tid == NT) some_s = some;
  }
  __syncthreads();
  const bool some    = some_s != 0;
  const float factor = some ? float(double(a.grad_loss[row]) * a.temperature) : 0.0f;
  T* g               = a.grad + row * a.ldg;
  const bool same    = same_phase(g, z);
  if (tid < NT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * NT + tid;
      if (j < part.n) {
        Words4 o;
#pragma unroll
        for (int e = 0; e < VE / 2; ++e) {
          const float2 f = up_pair<T>(raw[i], e);
          down_pair<T>(o, e, some ? make_float2(q(f.x) * factor, q(f.y) * factor) : make_float2(0.0f, 0.0f));
        }
        part.store(g + part.first, j, o, same);
      }
    }
  }
  __syncthreads();
  for (int j = tid; j < k && some; j += NT + 32) {
    const int t = id[j];
    float w;
    if (t >= part.token0 && t < part.token1 && listed_weight(id, logp, k, j, &w))
        g[t] = FloatIo<T>::down(factor * (q(zid[j]) - w));
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

template <typename Kernel, typename A>
inline cudaError_t launch_clusters(Kernel kern, const A& a, int64_t ctas, int size, int threads, size_t smem,
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

template <typename T, int NT, bool kEven>
inline cudaError_t launch_step_as(Args<T> a, int64_t most, int size, cudaStream_t stream)
{
  auto kern         = distill_step_kernel<T, NT, kEven>;
  const size_t smem = size_t(kStages) * NT * kStepNv * 16 + size_t(a.list.k) * 36 + NT * kStepNv * Vec16Of<T>::value / 8;
  a.per_cta         = int(ceil_div<int64_t>(most, size));
  cudaError_t e     = ensure_dynamic_smem(kern, smem);
  if (e != cudaSuccess) return e;
  const int64_t fit      = resident_clusters(kern, size, NT + 96, smem);
  const int64_t clusters = a.n_rows < fit ? a.n_rows : fit;
  return launch_clusters(kern, a, clusters * size, size, NT + 96, smem, stream);
}

template <typename T, int NT>
inline cudaError_t launch_step(const Args<T>& a, int64_t most, int size, cudaStream_t stream)
{
  const bool even = a.n_rows == 1 || uintptr_t(a.ldl) * sizeof(T) % 16 == 0;
  return even ? launch_step_as<T, NT, true>(a, most, size, stream) : launch_step_as<T, NT, false>(a, most, size, stream);
}

template <typename T, int NT, bool kGrad>
inline cudaError_t launch_stream(Args<T> a, int64_t most, int size, cudaStream_t stream)
{
  a.per_cta              = int(ceil_div<int64_t>(most, size));
  const size_t smem      = size_t(kStreamDepth) * NT * kStreamNv * 16 + size_t(a.list.k) * 12;
  const int64_t max_rows = int64_t(0x7fffffff) / size;
  cudaError_t e          = ensure_dynamic_smem(distill_stream_kernel<T, NT, kGrad>, smem);
  if (e != cudaSuccess) return e;
  for (int64_t r0 = 0; r0 < a.n_rows; r0 += max_rows) {
    const int64_t n = a.n_rows - r0 < max_rows ? a.n_rows - r0 : max_rows;
    e = launch_clusters(distill_stream_kernel<T, NT, kGrad>, rows_from(a, r0, n), n * size, size,
                                          NT + 32, smem, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Loss and gradient: a row is held by the CTAs of a cluster, 4096 vectors (64 KB) each; small vocabularies take small
// CTAs, and a row of more than 8 full ones is read twice, as are rows whose list does not fit beside the buffers
// (1024 x 262144 fp32: 488 us, 2.2 TB/s of one read and one write; 2048 x 32000 bf16 with 1000 entries: 2360 us, as every
// CTA compares its listed tokens with the whole list).
template <typename T>
inline cudaError_t launch_loss_and_grad(const Args<T>& a, cudaStream_t stream)
{
  const int64_t most = most_vectors(a);
  if (a.list.k > 800) return launch_stream<T, 256, true>(a, most, 8, stream);
  if (most <= 64 * kStepNv) return launch_step<T, 64>(a, most, 1, stream);
  if (most <= 256 * kStepNv) return launch_step<T, 256>(a, most, 1, stream);
  for (int size = 1; size <= 8; size *= 2)
    if (most <= int64_t(512) * kStepNv * size) return launch_step<T, 512>(a, most, size, stream);
  return launch_stream<T, 256, true>(a, most, 8, stream);
}

// Loss: rows are split over up to 8 CTAs, of at least four chunks each, while there are fewer than eight CTAs per SM
// (2048 x 131072 bf16: 115 us; split in two, with sixteen CTAs per SM, 120, and in four 138: what a CTA does before its
// first chunk and after its last one is not hidden by the others. The rule was swept there alone; by it 512 x 131072 fp32
// takes 52 us and 16384 x 32000 bf16 239, 1.25 and 1.47 times what their bytes take).
template <typename T>
inline cudaError_t launch_loss(const Args<T>& a, cudaStream_t stream)
{
  const int64_t most = most_vectors(a);
  if (most <= 128 * kStreamNv) return launch_stream<T, 128, false>(a, most, 1, stream);
  int size = 1;
  while (size < 8 && a.n_rows * size < 8 * int64_t(sm_count()) && most >= int64_t(256) * kStreamNv * 4 * size)
    size *= 2;
  return launch_stream<T, 256, false>(a, most, size, stream);
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
