// Distillation from a teacher's top logits: the loss of each row and its gradient.
//
// Row n of the student's logits z[V] against K teacher entries (id_k, t_k), with temperature tau and the
// soft cap c of the model's head (utils/model.py:204; c = 0: none):
//   s = c tanh(z / c) / tau  (or z / tau),   lse = log sum_j exp(s_j),   p = softmax over the row's entries of t / tau
//   loss = tau^2 sum_k p_k (log p_k - s[id_k] + lse)
//   d loss / dz_j = tau (exp(s_j - lse) - sum over k with id_k = j of p_k) (1 - tanh^2(z_j / c))
// An entry whose id is outside [0, V) is absent; a row without an entry above -inf has loss and gradient 0.
//
// Bound: HBM, with the issue slots and the special-function unit (16 results a cycle and SM) next: a logit takes
// one of it, one beyond the soft cap three. The loss reads a row once. Loss and gradient
// together read it once and write it once; the row waits between the two halves in shared memory:
//   - with a soft cap |s| <= c / tau, so the sums' reference is 0, no maximum is sought, and what waits is
//     exp(s) (1 - tanh^2), which the second half only multiplies by one factor of the row;
//   - without one a thread takes the maximum of its first values as its reference and looks for another only
//     when a sum leaves fp32's safe range; what waits are the loaded words, and their exponential is taken again.
// What it takes is bytes in flight and few instructions beside: a CTA is 128 threads, eight to an SM (one warp where
// rows are many and short), and each thread copies its own 16-byte slots into shared memory some batches ahead (loads to
// registers instead: a quarter more time; CTAs of 256 threads: 45 % more). Loss and gradient of 16,384 rows of 4,096
// soft-capped fp32 logits with 32 entries: 98 to 104 us, 5.2 to 5.5 TB/s; the loss alone 54 us, 5.0 TB/s, since a row's copies
// start and end with its CTA; 2,047 rows of 50,257 bf16 logits, the loss and then the gradient from its lse: 131 to 134
// us, 4.6 TB/s.
//
// A row too long for one CTA, or one of a few rows, is spread over a cluster of up to 8 CTAs whose sums meet
// through distributed shared memory, so no second launch or workspace is needed.
//
// The K entries are handled apart from the dense pass: every column is first written as if no entry
// named it, then the thread of an id's first entry rewrites that column with the sum over the entries
// of the same id, in entry order. Repeated ids are therefore added in the same order every time. Which entries repeat
// is found by a vote of a warp up to 32 entries and by a table of the ids beyond.
#include "operators.cuh"
#include "profile.cuh"
#include "ptx.cuh"

namespace noise {

constexpr int kDsSmThreads = 1024;       // threads an SM holds, in CTAs of 128 or 32
constexpr int kDsMaxK = 1024;
constexpr int kDsMaxCluster = 8;
constexpr int kDsRowBytes = 192 * 1024;  // shared memory that holds a CTA's part of a row, at most
// Slots of a batch, and batches a thread has in flight: on a ring, or as deep as it pays where the row stays. (Six batches
// of two everywhere: the gradient alone of 16,384 rows of 4,096 took 125 us instead of 100.)
template <bool kHold>
struct DsFlow {
  static constexpr int kBatch = kHold ? 1 : 2, kAhead = kHold ? 8 : 3;
  static constexpr int kSmallSlots = kHold ? 512 : 1536;  // a row that one warp takes, in slots
  static constexpr int ring(int threads) { return kHold ? 0 : kAhead * kBatch * threads * 16; }
};
constexpr int kDsTable = 2 * kDsMaxK * 8 + kDsMaxK * 2;  // the table of ids, at most

enum : int { kDsLoss = 0, kDsGrad = 1, kDsBoth = 2 };
// No soft cap; one whose c / tau keeps exp(s) within [e^-40, e^40], so that neither 2^30 of them nor their product with a
// slope of 1e-19 (23 caps) leaves fp32's normal range; any other.
enum : int { kCapNone = 0, kCapBound = 1, kCapFree = 2 };
constexpr float kDsBoundCap = 40.f;
constexpr double kDsFarLse = 1 << 29;  // lse in base 2 up to which 53 bits leave 24 behind the point

struct DistillParams {
  const void* logits;
  int64_t ld;
  const void* ids;
  int64_t ids_ld;
  int ids64;
  const void* teacher;
  int64_t teacher_ld;
  int teacher_type;
  const float* up;       // gradient of each row's loss (null: 1)
  const double* lse_in;  // gradient from a saved lse
  float* loss;
  double* lse;
  void* grad;
  int64_t grad_ld;
  int64_t rows;
  int V, K, parts, shift;  // parts: CTAs per row, 2^shift
  int id_at;             // bytes of dynamic shared memory before the entries' ids
  int table;             // places of the table of ids, a power of two of at least 2 K
  float tau, cap, inv_tau, inv_cap;
};

// A slot is 16 bytes of a row, counted from the 16-byte boundary at or before its first element, so the
// first and last slots may be partial.
template <typename E>
struct DsSlot {
  static constexpr int kN = 16 / sizeof(E);
};

template <typename E>
__device__ __forceinline__ void slot_values(const uint4& w, float2 (&v)[DsSlot<E>::kN / 2]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(E) == 4) {
    v[0] = make_float2(__uint_as_float(u[0]), __uint_as_float(u[1]));
    v[1] = make_float2(__uint_as_float(u[2]), __uint_as_float(u[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = unpack2<E>(u[i]);
  }
}

template <typename E>
__device__ __forceinline__ uint4 slot_pack(const float2 (&v)[DsSlot<E>::kN / 2]) {
  if constexpr (sizeof(E) == 4)
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  else
    return make_uint4(pack2<E>(v[0].x, v[0].y), pack2<E>(v[1].x, v[1].y), pack2<E>(v[2].x, v[2].y),
                      pack2<E>(v[3].x, v[3].y));
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 ex2_pair(float2 x) { return make_float2(ex2_approx(x.x), ex2_approx(x.y)); }

// tanh to about 2 ulp and its slope 1 - tanh^2 to about (4 |x| + 8) half ulp. Up to |x| = 1 from a polynomial x + x^3 Q(x^2): Q is a least-squares fit of degree 6 at Chebyshev
// nodes, off by 1.3e-8 of tanh, 8.2e-8 as fp32 takes it. Beyond, where 1 - e no longer cancels, from e = exp(-2 |x|): (1 - e) / (1 + e), and the slope
// as 4 e / (1 + e)^2, since 1 - tanh^2 would have lost all its digits at |x| = 9. Logits within the soft cap, nearly all
// of a trained model's, so take no special function for their tanh.
__device__ __forceinline__ float2 tanh_near(float2 x) {
  const float2 u = __fmul2_rn(x, x);
  float2 q = __ffma2_rn(both(-3.552270937e-4f), u, both(2.289985307e-3f));
  q = __ffma2_rn(q, u, both(-7.930326276e-3f));
  q = __ffma2_rn(q, u, both(2.147581428e-2f));
  q = __ffma2_rn(q, u, both(-5.387599394e-2f));
  q = __ffma2_rn(q, u, both(1.333228201e-1f));
  q = __ffma2_rn(q, u, both(-3.333329260e-1f));
  return __ffma2_rn(__fmul2_rn(x, u), q, x);
}
__device__ __forceinline__ float2 slope_near(float2 th) {
  return __ffma2_rn(make_float2(-th.x, -th.y), th, both(1.f));
}
__device__ __forceinline__ float tanh_far(float x, float& slope) {
  const float e = ex2_approx(fabsf(x) * -2.8853900817779268f), r = rcp_approx(1.f + e);
  slope = 4.f * e * r * r;
  return copysignf((1.f - e) * r, x);
}
__device__ __forceinline__ float2 ds_tanh(float2 x, float2& slope) {
  float2 th = tanh_near(x);
  slope = slope_near(th);
  if (!(fabsf(x.x) <= 1.f)) th.x = tanh_far(x.x, slope.x);
  if (!(fabsf(x.y) <= 1.f)) th.y = tanh_far(x.y, slope.y);
  return th;
}

// A reference m and the sum of 2^(scale (. - m)); an empty or all -inf set is (-inf, 0). The difference is taken
// before the scale, so that values near the type's lowest do not turn into -inf.
struct MaxSum {
  float m, s;
  __device__ __forceinline__ void join(float om, float os, float scale = 1.f) {
    const float top = fmaxf(m, om);
    const float base = top == -INFINITY ? 0.f : top;
    s = (m == -INFINITY ? s : s * exp2f((m - base) * scale)) + (om == -INFINITY ? os : os * exp2f((om - base) * scale));
    m = top;
  }
};

template <typename E, int kMode, int kCap, int kDsThreads>
__global__ void __launch_bounds__(kDsThreads, kDsSmThreads / kDsThreads) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int N = DsSlot<E>::kN;
  constexpr bool kHold = kMode == kDsBoth;  // the row stays in shared memory
  constexpr bool kBound = kCap == kCapBound;
  constexpr int kDsBatch = DsFlow<kHold>::kBatch, kDsAhead = DsFlow<kHold>::kAhead;
  constexpr float kLog2e = 1.4426950408889634f;
  // the row's slots (kHold; with a bound soft cap N / 4 planes of fp32 per slot), or a ring of batches in flight
  extern __shared__ uint4 hold[];
  int* s_id = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(hold) + p.id_at);  // [K]
  constexpr int kDsWarps = kDsThreads / 32;
  __shared__ float red[5][kDsWarps];
  __shared__ float2 part;  // this CTA's (m, s), read by the cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x >> p.shift;
  const int rank = blockIdx.x & (p.parts - 1);
  const E* z = reinterpret_cast<const E*>(p.logits) + row * p.ld;
  const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(E));
  const E* z0 = z - phase;  // 16-byte aligned; element e of the row is z0[e + phase]
  const int slots = (p.V + phase + N - 1) / N;
  const int share = (slots + p.parts - 1) >> p.shift;
  const int begin = min(slots, rank * share), end = min(slots, begin + share);
  const float inv_tau = p.inv_tau, inv_cap = p.inv_cap;
  // s in base 2 is scale * v, with v = z, or tanh(z / c). References are values of v, and v's difference from one is
  // taken before the scale: a row whose every logit is a mask's -1e30, or the type's lowest value, then has the sums of a
  // row of equal logits, where scale * v has lost them or is -inf.
  const float scale = (kCap ? p.cap : 1.f) * inv_tau * kLog2e;

  // This CTA's whole slots, and its share of the row's at most two partial ones, an element a thread: the head's by
  // threads 0 .. 6, the tail's by threads 8 .. 14.
  const int head = (N - phase) % N, tail = head + (p.V - head > 0 ? (p.V - head) / N * N : 0);  // [head, tail): whole slots
  const int skip = phase ? 1 : 0;
  const int first = max(begin, skip), last = min(end, skip + (tail - head) / N);
  const bool has_head = phase && begin == 0 && end > 0, has_tail = tail < p.V && end == slots && end > begin;
  int edge = -1;
  if (has_head && tid < min(head, p.V)) edge = tid;
  if (has_tail && tid >= 8 && tid - 8 < p.V - max(tail, head)) edge = max(tail, head) + tid - 8;
  const float z_edge = edge >= 0 ? to_f32(z[edge]) : 0.f;
  const uint4* z16 = reinterpret_cast<const uint4*>(z0);
  // f(batch of slots, its first slot, how many) for this thread's slots first + tid, + kDsThreads, ..: each thread
  // copies its own slots into its own places, kDsAhead batches ahead, on a ring or (kHold) to where they stay
  constexpr uint32_t kPitch = kDsThreads * 16, kBatchBytes = kDsBatch * kPitch, kWrap = kHold ? 0u : kDsAhead * kBatchBytes;
  const uint32_t own = (kHold ? first - begin : 0) * 16 + tid * 16;
  const uint4* source = z16 + first + tid;
  int coming = last - first - tid;  // slots from this thread's next one on
  uint32_t into = own;
  auto advance = [&](uint32_t& at) {
    at += kBatchBytes;
    if (!kHold && at >= kWrap) at -= kWrap;
  };
  const uint32_t hold0 = smem_u32(hold);
  auto issue = [&] {
#pragma unroll
    for (int u = 0; u < kDsBatch; ++u)
      if (u * kDsThreads < coming) cp_async16(hold0 + into + u * kPitch, source + u * kDsThreads);
    cp_async_commit();
    source += kDsBatch * kDsThreads, coming -= kDsBatch * kDsThreads;
    advance(into);
  };
  auto start = [&] {
#pragma unroll
    for (int i = 0; i < kDsAhead - 1; ++i) issue();
  };
  auto sweep = [&](auto&& f) {
    uint32_t from = own;
    for (int slot = first + tid; slot < last; slot += kDsBatch * kDsThreads) {
      issue();
      cp_async_wait<kDsAhead - 1>();
      uint4 w[kDsBatch];
      const int count = min(kDsBatch, (last - slot + kDsThreads - 1) / kDsThreads);
#pragma unroll
      for (int u = 0; u < kDsBatch; ++u)
        if (u < count) w[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(hold) + from + u * kPitch);
      advance(from);
      f(w, slot, count);
    }
  };
  start();
  // v of a slot and, with a soft cap, its slope d v / d (z / c); the same numbers on either way
  auto values = [&](float2 (&v)[N / 2], float2 (&slope)[N / 2]) {
    if (!kCap) return;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = __fmul2_rn(v[i], both(inv_cap)), top = max3(top, fabsf(v[i].x), fabsf(v[i].y));
    if (top <= 1.f) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) v[i] = tanh_near(v[i]), slope[i] = slope_near(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) v[i] = ds_tanh(v[i], slope[i]);
    }
  };
  auto value1 = [&](float x, float& slope) {
    if (!kCap) return x;
    float2 two;
    const float v = ds_tanh(both(x * inv_cap), two).x;
    slope = two.x;
    return v;
  };
  float unused;

  // Entry k: its id (-1: absent) and logit. A thread keeps its first one, k = tid, in registers from the start.
  auto entry = [&](int k, int& id) {
    const int64_t at = row * p.ids_ld + k, tt = row * p.teacher_ld + k;
    const int64_t i = p.ids64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + at)
                              : (int64_t)__ldg(reinterpret_cast<const int*>(p.ids) + at);
    const float t = p.teacher_type == NOISE_FP32   ? reinterpret_cast<const float*>(p.teacher)[tt]
                    : p.teacher_type == NOISE_BF16 ? to_f32(reinterpret_cast<const __nv_bfloat16*>(p.teacher)[tt])
                                                   : to_f32(reinterpret_cast<const __half*>(p.teacher)[tt]);
    const bool have = i >= 0 && i < p.V;
    id = have ? (int)i : -1;
    return have ? t : -INFINITY;
  };
  int id0 = -1;
  float t0 = -INFINITY;
  if (tid < p.K) t0 = entry(tid, id0);
  // the teacher's maximum and mass: p_k = 2^(t_scale (t_k - max)) / mass, 0 for absent entries. The warps' parts of them
  // are formed here, while the row's first copies are on their way.
  const float t_scale = inv_tau * kLog2e;
  if (warp * 32 < p.K) {
    MaxSum c{t0, t0 == -INFINITY ? 0.f : 1.f};
    if (kMode != kDsLoss && tid < p.K) s_id[tid] = id0;
    for (int k = tid + kDsThreads; k < p.K; k += kDsThreads) {
      int id;
      const float t = entry(k, id);
      if (kMode != kDsLoss) s_id[k] = id;
      c.join(t, t == -INFINITY ? 0.f : 1.f, t_scale);
    }
    float top = c.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float mass = c.m == -INFINITY ? c.s : c.s * exp2f((c.m - top) * t_scale);
#pragma unroll
    for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    if (lane == 0) red[2][warp] = top, red[3][warp] = mass;
  }
  const float z_id = id0 >= 0 ? to_f32(z[id0]) : 0.f;

  MaxSum a{kBound ? 0.f : -INFINITY, 0.f};
  if constexpr (kMode != kDsGrad) {
    // one slot's sum under the reference as it stands
    auto add = [&](const uint4& w, int slot, float2& sum) {
      float2 v[N / 2], slope[N / 2];
      slot_values<E>(w, v);
      values(v, slope);
      if constexpr (kBound) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 e = ex2_pair(__fmul2_rn(v[i], both(scale)));
          sum = __fadd2_rn(sum, e);
          if (kHold) v[i] = __fmul2_rn(e, slope[i]);
        }
        if constexpr (kHold) {
#pragma unroll
          for (int i = 0; i < N / 4; ++i)
            reinterpret_cast<float4*>(hold)[i * share + slot - begin] =
                make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
        }
      } else {
        const float2 off = both(a.m == -INFINITY ? 0.f : -a.m);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) sum = __fadd2_rn(sum, ex2_pair(__fmul2_rn(__fadd2_rn(v[i], off), both(scale))));
      }
    };
    // a reference that the slots from `slot` on, `count` of them, do not overflow
    auto raise = [&](int slot, int count) {
      float m = -INFINITY;
#pragma unroll 1
      for (int e = slot * N - phase; count; e += kDsThreads * N, --count)
#pragma unroll 1
        for (int i = 0; i < N; ++i) m = fmaxf(m, value1(to_f32(z[e + i]), unused));
      if (m > a.m) a.s = a.m == -INFINITY ? a.s : a.s * exp2f((a.m - m) * scale), a.m = m;
    };
    auto take = [&](const uint4* w, int slot, int count) {
      if (!kBound && a.m == -INFINITY) raise(slot, count);
      float2 sum = both(0.f);
#pragma unroll
      for (int u = 0; u < kDsBatch; ++u)
        if (u < count) add(w[u], slot + u * kDsThreads, sum);
      if (!kBound && !(sum.x + sum.y < 1e30f)) {
        raise(slot, count);
        sum = both(0.f);
#pragma unroll
        for (int u = 0; u < kDsBatch; ++u)
          if (u < count) add(w[u], slot + u * kDsThreads, sum);
      }
      a.s += sum.x + sum.y;
    };
    sweep(take);
    if (edge >= 0) {
      const float x = value1(z_edge, unused);
      if (kBound) a.s += ex2_approx(x * scale);
      else a.join(x, x == -INFINITY ? 0.f : 1.f, scale);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (kMode == kDsGrad) break;
    const float os = __shfl_xor_sync(0xffffffffu, a.s, o);
    if (kBound) a.s += os;
    else a.join(__shfl_xor_sync(0xffffffffu, a.m, o), os, scale);
  }
  if (lane == 0) red[0][warp] = a.m, red[1][warp] = a.s;
  __syncthreads();
  MaxSum c{red[2][0], red[3][0]};
#pragma unroll
  for (int w = 1; w < kDsWarps; ++w)
    if (w * 32 < p.K) c.join(red[2][w], red[3][w], t_scale);
  const float top = c.m, mass = c.s;
  const bool empty = mass == 0.f;
  const float inv_mass = 1.0f / mass;
  if constexpr (kMode != kDsGrad) {
    a = MaxSum{red[0][0], red[1][0]};
#pragma unroll
    for (int w = 1; w < kDsWarps; ++w) {
      if (kBound) a.s += red[1][w];
      else a.join(red[0][w], red[1][w], scale);
    }
    if (p.parts > 1) {
      if (tid == 0) part = make_float2(a.m, a.s);
      cluster_sync();
      MaxSum all{-INFINITY, 0.f};
      for (int r = 0; r < p.parts; ++r) {
        const uint32_t at = cluster_addr(&part, (uint32_t)r);
        all.join(__uint_as_float(ld_cluster_u32(at)), __uint_as_float(ld_cluster_u32(at + 4)), scale);
      }
      a = all;
      cluster_sync();  // no CTA of the cluster leaves while another reads its part
    }
  }

  // the loss's terms, added up behind the dense gradient
  if (kMode != kDsGrad && rank == 0 && warp * 32 < p.K) {
    const float log_mass = logf(mass), log_sum = logf(a.s);
    float l = 0.f;
    auto term = [&](int id, float t, float x) {
      const float d = (t - top) * inv_tau, pk = exp2f((t - top) * t_scale) * inv_mass;
      // tau times the term, with lse - s from the difference of v and the reference: finite wherever the loss is
      if (id >= 0 && pk != 0.f)
        l += pk * (p.tau * ((d - log_mass) + log_sum) - (value1(x, unused) - a.m) * (kCap ? p.cap : 1.f));
    };
    if (tid < p.K) term(id0, t0, z_id);
    for (int k = tid + kDsThreads; k < p.K; k += kDsThreads) {
      int id;
      const float t = entry(k, id);
      if (id >= 0) term(id, t, to_f32(z[id]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[4][warp] = l;
  }
  auto finish = [&] {  // after a barrier
    if (kMode == kDsGrad || rank != 0 || tid != 0) return;
    float l = red[4][0];
#pragma unroll
    for (int w = 1; w < kDsWarps; ++w)
      if (w * 32 < p.K) l += red[4][w];
    p.loss[row] = empty ? 0.f : p.tau * l;
    // in 64 bits: the gradient's exponentials have the error of this number in common
    if (p.lse) p.lse[row] = 0.6931471805599453094 * ((double)a.m * (double)scale + log2((double)a.s));
  };

  if constexpr (kMode != kDsLoss) {
    E* g = reinterpret_cast<E*>(p.grad) + row * p.grad_ld;
    const bool same = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(E)) == phase;
    const float up = empty ? 0.f : p.tau * (p.up ? __ldg(p.up + row) : 1.0f);
    // softmax(s) is 2^(scale (v - ref) - low) * factor
    float ref = a.m, low = 0.f, factor = 1.f / a.s;
    if constexpr (kMode == kDsGrad) {
      const double lse2 = p.lse_in[row] * 1.4426950408889634074;
      ref = (float)(lse2 / (double)scale), low = (float)(lse2 - (double)ref * (double)scale), factor = 1.f;
      if (!isfinite(ref)) ref = 0.f, low = (float)lse2;
      if (isfinite(lse2) && !(fabs(lse2) < kDsFarLse) && !empty) {
        // so far out that lse in 64 bits has not the 24 bits left that the gradient needs: the row's sum once more, by
        // every CTA of the row for itself
        MaxSum far{-INFINITY, 0.f};
        for (int e = tid; e < p.V; e += kDsThreads) {
          const float v = value1(to_f32(z[e]), unused);
          far.join(v, v == -INFINITY ? 0.f : 1.f, scale);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const float os = __shfl_xor_sync(0xffffffffu, far.s, o);
          far.join(__shfl_xor_sync(0xffffffffu, far.m, o), os, scale);
        }
        __syncthreads();  // red's last readers are done
        if (lane == 0) red[0][warp] = far.m, red[1][warp] = far.s;
        __syncthreads();
        far = MaxSum{red[0][0], red[1][0]};
#pragma unroll
        for (int w = 1; w < kDsWarps; ++w) far.join(red[0][w], red[1][w], scale);
        ref = far.m, low = 0.f, factor = 1.f / far.s;
      }
    }
    // gradient at a column from its logit, with the entries' mass pj there
    auto column = [&](float x, float pj) {
      float slope;
      const float v = value1(x, slope);
      const float d = up * fmaf(ex2_approx(fmaf(v - ref, scale, -low)), factor, -pj);
      return kCap ? d * slope : d;
    };
    uint4* g16 = reinterpret_cast<uint4*>(g - phase);
    auto write = [&](int slot, const float2 (&v)[N / 2]) {
      if (same) {
        __stcs(g16 + slot, slot_pack<E>(v));
      } else {
        E* at = g + slot * N - phase;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) at[2 * i] = from_f32<E>(v[i].x), at[2 * i + 1] = from_f32<E>(v[i].y);
      }
    };
    if (empty) {
      cp_async_wait<0>();  // the gradient alone has not taken its first copies: they land before the CTA leaves
      float2 v[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) v[i] = both(0.f);
      for (int slot = first + tid; slot < last; slot += kDsThreads) write(slot, v);
      if (edge >= 0) g[edge] = from_f32<E>(0.f);
      __syncthreads();
      finish();
      return;
    }
    const float2 gain = both(up * factor);
    auto spread = [&](const uint4& w, int slot) {
      float2 v[N / 2];
      if constexpr (kHold && kBound) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
          const float4 x = reinterpret_cast<const float4*>(hold)[i * share + slot - begin];
          v[2 * i] = __fmul2_rn(make_float2(x.x, x.y), gain), v[2 * i + 1] = __fmul2_rn(make_float2(x.z, x.w), gain);
        }
      } else {
        float2 slope[N / 2];
        slot_values<E>(w, v);
        values(v, slope);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 away = __fadd2_rn(v[i], both(-ref));
          const float2 y = kMode == kDsGrad ? __ffma2_rn(away, both(scale), both(-low)) : __fmul2_rn(away, both(scale));
          v[i] = __fmul2_rn(ex2_pair(y), gain);
          if (kCap) v[i] = __fmul2_rn(v[i], slope[i]);
        }
      }
      write(slot, v);
    };
    if constexpr (kMode == kDsGrad) {
      sweep([&](const uint4* w, int slot, int count) {
#pragma unroll
        for (int u = 0; u < kDsBatch; ++u)
          if (u < count) spread(w[u], slot + u * kDsThreads);
      });
    } else {
#pragma unroll 4
      for (int slot = first + tid; slot < last; slot += kDsThreads)
        spread(kBound ? make_uint4(0u, 0u, 0u, 0u) : hold[slot - begin], slot);
    }
    if (edge >= 0) g[edge] = from_f32<E>(column(z_edge, 0.f));
    __syncthreads();  // the dense stores of this CTA come before its entries' stores
    finish();
    const int e0 = begin * N - phase, e1 = min(p.V, end * N - phase);
    auto here = [&](int id) { return id >= e0 && id < e1 && id >= 0; };
    auto rewrite = [&](int k, int id, bool again) {
      int other;
      float pj = exp2f(((k == tid ? t0 : entry(k, other)) - top) * t_scale) * inv_mass;
      if (again)
        for (int i = k + 1; i < p.K; ++i)
          if (s_id[i] == id) pj += exp2f((entry(i, other) - top) * t_scale) * inv_mass;
      g[id] = from_f32<E>(column(k == tid ? z_id : to_f32(z[id]), pj));
    };
    if (p.K <= 32) {  // equal ids by a vote of one warp
      if (warp == 0) {
        const int id = lane < p.K ? s_id[lane] : -1;
        const uint32_t equal = __match_any_sync(0xffffffffu, id);
        if (here(id) && (equal & ((1u << lane) - 1u)) == 0) rewrite(lane, id, (equal >> lane) > 1u);
      }
    } else {
      // by a table of the ids, over the memory that the row has left: a place's id (its sign bit: named again), its
      // first entry, and each entry's place. Where an id lies depends on timing; what the table says of it does not.
      int* t_id = reinterpret_cast<int*>(hold);
      int* t_first = t_id + p.table;
      uint16_t* at = reinterpret_cast<uint16_t*>(t_first + p.table);
      for (int i = tid; i < p.table; i += kDsThreads) t_id[i] = -1, t_first[i] = kDsMaxK;
      __syncthreads();
      for (int k = tid; k < p.K; k += kDsThreads) {
        const int id = s_id[k];
        if (!here(id)) continue;
        uint32_t h = (uint32_t)id * 2654435769u >> 16;  // the multiplier of Fibonacci hashing, 2^32 / golden ratio
        while (true) {  // at most half of the places are taken
          h &= p.table - 1;
          const int was = atomicCAS(&t_id[h], -1, id);
          if (was == -1 || was == id) break;
          ++h;
        }
        atomicMin(&t_first[h], k);
        at[k] = (uint16_t)h;
      }
      __syncthreads();
      for (int k = tid; k < p.K; k += kDsThreads)
        if (here(s_id[k]) && t_first[at[k]] != k) t_id[at[k]] = s_id[k] | (int)0x80000000;
      __syncthreads();
      for (int k = tid; k < p.K; k += kDsThreads)
        if (here(s_id[k]) && t_first[at[k]] == k) rewrite(k, s_id[k], t_id[at[k]] < 0);
    }
  } else {
    __syncthreads();
    finish();
  }
}

int device_sm_count();

// Bytes of shared memory that `parts` CTAs each need to hold their part of a row.
static int64_t ds_hold_bytes(int V, int elem, bool planes, int parts) {
  const int n = 16 / elem;
  const int64_t slots = ((int64_t)V + 2 * n - 1) / n;
  const int64_t share = (slots + parts - 1) / parts;
  return share * (planes ? 4 * n : 16);
}

template <typename E, int kMode, int kCap, int kThreads>
static int launch_distill(DistillParams& p, int parts, int smem, cudaStream_t s) {
  static KernelOptIn opt_in;
  constexpr int kMost = (kMode == kDsBoth ? kDsRowBytes : kDsTable) + kDsMaxK * 4;
  if (!opt_in(distill_kernel<E, kMode, kCap, kThreads>, kMost)) return kStatusLaunchFailed;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)parts, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * parts)), cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem, cfg.stream = s;
  cfg.attrs = &attr, cfg.numAttrs = kMode != kDsGrad && parts > 1;  // the gradient's CTAs share nothing
  LaunchScope scope(kKindLoss, s);
  if (cudaLaunchKernelEx(&cfg, distill_kernel<E, kMode, kCap, kThreads>, p) != cudaSuccess) {
    cudaGetLastError();
    return kStatusLaunchFailed;
  }
  return kStatusOk;
}

template <typename E, int kMode, int kCap>
static int launch_distill(DistillParams& p, cudaStream_t s) {
  // CTAs per row: until every SM has two, of at least four slots a thread; more where a row must fit shared memory.
  // (Splitting 2,047 rows of 50,257 over clusters of 4 to even out the last CTAs took 188 us instead of 139.)
  const int64_t slots = ((int64_t)p.V + DsSlot<E>::kN - 1) / DsSlot<E>::kN;
  const int64_t want = 2 * (int64_t)device_sm_count();
  int parts = 1;
  while (parts < kDsMaxCluster && p.rows * parts < want && slots / (2 * parts) >= 4 * 128) parts *= 2;
  if (kMode == kDsBoth)
    while (parts < kDsMaxCluster && ds_hold_bytes(p.V, sizeof(E), kCap == kCapBound, parts) > kDsRowBytes / 4) parts *= 2;
  // CTAs of one warp where there are more rows than fit the GPU in CTAs of four and a row is short: the steps that come
  // once a row then wait for nothing but themselves. Loss, gradient alone and both in us, four warps against one: 9,678
  // rows of 258 slots 51, 33, 57 / 29, 16, 37; 16,384 of 1,024 76, 98, 102 / 64, 88, 107; 6,000 of 1,251 53, 47, 70 /
  // 43, 43, 90; 4,000 of 2,048 49, 57, 92 / 51, 59, 92. The row that stays in shared memory wants more threads a CTA.
  const bool small = parts == 1 && p.rows > 8 * (int64_t)device_sm_count() && p.K <= 256 &&
                     slots <= DsFlow<kMode == kDsBoth>::kSmallSlots;
  int64_t smem = DsFlow<kMode == kDsBoth>::ring(small ? 32 : 128);
  static_assert(DsFlow<false>::ring(128) <= kDsTable, "the opt-in covers the ring");
  if (kMode == kDsBoth) smem = ds_hold_bytes(p.V, sizeof(E), kCap == kCapBound, parts);
  if (smem > kDsRowBytes || p.rows * parts > INT32_MAX) return kStatusUnsupported;
  if (kMode != kDsLoss) {
    if (p.K > 32) {
      for (p.table = 64; p.table < 2 * p.K;) p.table *= 2;
      smem = max(smem, (int64_t)p.table * 8 + (p.K * 2 + 15) / 16 * 16);
    }
    p.id_at = (int)smem, smem += (p.K + 3) / 4 * 16;
  }
  p.parts = parts;
  for (p.shift = 0; 1 << p.shift < parts;) ++p.shift;
  p.inv_tau = 1.0f / p.tau, p.inv_cap = kCap ? 1.0f / p.cap : 0.f;
  return small ? launch_distill<E, kMode, kCap, 32>(p, parts, (int)smem, s)
               : launch_distill<E, kMode, kCap, 128>(p, parts, (int)smem, s);
}

template <typename E, int kMode>
static int launch_distill_cap(DistillParams& p, cudaStream_t s) {
  if (p.cap == 0.f) return launch_distill<E, kMode, kCapNone>(p, s);
  return p.cap / p.tau <= kDsBoundCap ? launch_distill<E, kMode, kCapBound>(p, s) : launch_distill<E, kMode, kCapFree>(p, s);
}

template <typename E>
static int launch_distill_mode(DistillParams& p, int mode, cudaStream_t s) {
  return mode == kDsLoss ? launch_distill_cap<E, kDsLoss>(p, s)
                         : mode == kDsGrad ? launch_distill_cap<E, kDsGrad>(p, s) : launch_distill_cap<E, kDsBoth>(p, s);
}

}  // namespace noise

using namespace noise;

extern "C" int64_t noise_distill_max_vocab(int dtype, int softcap) {
  const int elem = dtype == NOISE_FP32 ? 4 : 2;
  const int64_t per_slot = softcap ? 64 / elem : 16;
  return ((int64_t)kDsMaxCluster * (kDsRowBytes / per_slot) - 2) * (16 / elem);
}

extern "C" int noise_distill(const NoiseDistill* a, void* stream) {
  if (!a || a->N < 0 || a->V < 1 || a->K < 1 || !(a->temperature > 0.f) || !(a->softcap >= 0.f))
    return kStatusBadArgument;
  if (!a->logits || !a->ids || !a->teacher || a->ld < a->V || a->ids_ld < a->K || a->teacher_ld < a->K)
    return kStatusBadArgument;
  if (a->K > kDsMaxK || a->V > (1 << 30)) return kStatusUnsupported;
  const int mode = a->lse_in ? kDsGrad : a->grad ? kDsBoth : kDsLoss;
  if (mode == kDsGrad && !a->grad) return kStatusBadArgument;
  if (mode != kDsGrad && !a->loss) return kStatusBadArgument;
  if (a->grad && a->grad_ld < a->V) return kStatusBadArgument;
  if (a->N == 0) return kStatusOk;
  if (a->grad) {  // the entries' columns are read again after the dense gradient is written
    const uint64_t elem = a->dtype == NOISE_FP32 ? 4 : 2;
    const uint64_t z = reinterpret_cast<uint64_t>(a->logits), g = reinterpret_cast<uint64_t>(a->grad);
    const uint64_t zn = ((a->N - 1) * a->ld + a->V) * elem, gn = ((a->N - 1) * a->grad_ld + a->V) * elem;
    if (z < g + gn && g < z + zn) return kStatusBadArgument;
  }
  DistillParams p{};
  p.logits = a->logits, p.ld = a->ld, p.ids = a->ids, p.ids_ld = a->ids_ld, p.ids64 = a->ids_int64;
  p.teacher = a->teacher, p.teacher_ld = a->teacher_ld, p.teacher_type = a->teacher_dtype;
  p.up = a->dloss, p.lse_in = a->lse_in, p.loss = a->loss, p.lse = a->lse, p.grad = a->grad, p.grad_ld = a->grad_ld;
  p.rows = a->N, p.V = a->V, p.K = a->K, p.tau = a->temperature, p.cap = a->softcap;
  if (p.teacher_type != NOISE_FP32 && p.teacher_type != NOISE_BF16 && p.teacher_type != NOISE_FP16)
    return kStatusUnsupported;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case NOISE_FP32: return launch_distill_mode<float>(p, mode, s);
    case NOISE_BF16: return launch_distill_mode<__nv_bfloat16>(p, mode, s);
    case NOISE_FP16: return launch_distill_mode<__half>(p, mode, s);
  }
  return kStatusUnsupported;
}
