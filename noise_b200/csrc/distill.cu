// Distillation from a teacher's top logits: the loss of each row and its gradient.
//
// Row n of the student's logits z[V] against K teacher entries (id_k, t_k), with temperature tau and the
// soft cap c of the model's head (utils/model.py:204; c = 0: none):
//   s = c tanh(z / c) / tau  (or z / tau),   lse = log sum_j exp(s_j),   p = softmax over the row's entries of t / tau
//   loss = tau^2 sum_k p_k (log p_k - s[id_k] + lse)
//   d loss / dz_j = tau (exp(s_j - lse) - sum over k with id_k = j of p_k) (1 - tanh^2(z_j / c))
// An entry whose id is outside [0, V) is absent; a row without an entry above -inf has loss and gradient 0.
//
// Bound: HBM. The loss reads a row once, with a running maximum and sum in each thread. Loss and gradient
// together read it once and write it once: the row's values stay in shared memory between the two
// halves of the work, s as fp32 where the soft cap made it costly, the loaded words otherwise. A row
// too long for one CTA, or one of a few rows, is spread over a cluster of up to 8 CTAs whose maxima and
// sums meet through distributed shared memory, so no second launch or workspace is needed.
//
// The K entries are handled apart from the dense pass: every column is first written as if no entry
// named it, then the thread of an id's first entry rewrites that column with the sum over the entries
// of the same id, in entry order. Repeated ids are therefore added in the same order every time.
#include "operators.cuh"
#include "profile.cuh"
#include "ptx.cuh"

namespace noise {

constexpr int kDsThreads = 256, kDsWarps = kDsThreads / 32;
constexpr int kDsMaxK = 1024;
constexpr int kDsMaxCluster = 8;
constexpr int kDsRowBytes = 192 * 1024;  // shared memory that holds a CTA's part of a row, at most

enum : int { kDsLoss = 0, kDsGrad = 1, kDsBoth = 2 };

struct DistillParams {
  const void* logits;
  int64_t ld;
  const void* ids;
  int64_t ids_ld;
  int ids64;
  const void* teacher;
  int64_t teacher_ld;
  int teacher_type;
  const float* up;      // gradient of each row's loss (null: 1)
  const float* lse_in;  // gradient from a saved lse
  float* loss;
  float* lse;
  void* grad;
  int64_t grad_ld;
  int64_t rows;
  int V, K, parts;      // parts: CTAs per row
  float tau, cap;
};

// A slot is 16 bytes of a row, counted from the 16-byte boundary at or before its first element, so the
// first and last slots may be partial.
template <typename E>
struct DsSlot {
  static constexpr int kN = 16 / sizeof(E);
};

template <typename E>
__device__ __forceinline__ void slot_values(const uint4& w, float (&v)[DsSlot<E>::kN]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<E>(u[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

template <typename E>
__device__ __forceinline__ uint4 slot_pack(const float (&v)[DsSlot<E>::kN]) {
  if constexpr (sizeof(E) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7]));
}

// exp of a difference that is <= 0 up to rounding.
__device__ __forceinline__ float ds_exp(float x) { return expf(x); }

// A running maximum m and the sum of exp(. - m); an empty or all -inf set is (-inf, 0).
struct MaxSum {
  float m, s;
  __device__ __forceinline__ void join(float om, float os) {
    const float top = fmaxf(m, om);
    const float base = top == -INFINITY ? 0.f : top;
    s = (m == -INFINITY ? s : s * ds_exp(m - base)) + (om == -INFINITY ? os : os * ds_exp(om - base));
    m = top;
  }
};

template <typename E, int kMode, bool kCap>
__global__ void __launch_bounds__(kDsThreads) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int N = DsSlot<E>::kN;
  constexpr bool kHold = kMode == kDsBoth;  // the row stays in shared memory
  extern __shared__ uint4 hold[];           // raw slots, or with a soft cap N / 4 planes of s
  __shared__ int s_id[kDsMaxK];
  __shared__ float s_p[kDsMaxK];
  __shared__ float red[2][kDsWarps];
  __shared__ float2 part;  // this CTA's (m, s), read by the cluster
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / p.parts;
  const int rank = blockIdx.x - (int)(row * p.parts);
  const E* z = reinterpret_cast<const E*>(p.logits) + row * p.ld;
  const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(E));
  const E* z0 = z - phase;  // 16-byte aligned; element e of the row is z0[e + phase]
  const int slots = (p.V + phase + N - 1) / N;
  const int share = (slots + p.parts - 1) / p.parts;
  const int begin = min(slots, rank * share), end = min(slots, begin + share);
  const float inv_tau = 1.0f / p.tau, inv_cap = kCap ? 1.0f / p.cap : 0.f;
  const float s_of = kCap ? p.cap * inv_tau : inv_tau;  // s = s_of * tanh(z / c), or s_of * z

  auto load = [&](int slot) {
    if (slot * N >= phase && (slot + 1) * N <= p.V + phase)
      return __ldcs(reinterpret_cast<const uint4*>(z0) + slot);
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = slot * N + i - phase;
      v[i] = e >= 0 && e < p.V ? to_f32(z[e]) : -INFINITY;
    }
    return slot_pack<E>(v);
  };
  auto to_s = [&](float x) { return kCap ? s_of * tanhf(x * inv_cap) : s_of * x; };

  // the teacher's entries: p_k = exp((t_k - max) / tau) / mass, 0 for absent ones. The maximum is taken off
  // before the division, so that entries at the type's lowest value do not turn into -inf.
  float top = -INFINITY;
  for (int k = tid; k < p.K; k += kDsThreads) {
    const int64_t at = row * p.ids_ld + k;
    const int64_t id = p.ids64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + at)
                               : (int64_t)__ldg(reinterpret_cast<const int*>(p.ids) + at);
    const int64_t tt = row * p.teacher_ld + k;
    float t = p.teacher_type == NOISE_FP32   ? reinterpret_cast<const float*>(p.teacher)[tt]
              : p.teacher_type == NOISE_BF16 ? to_f32(reinterpret_cast<const __nv_bfloat16*>(p.teacher)[tt])
                                             : to_f32(reinterpret_cast<const __half*>(p.teacher)[tt]);
    const bool have = id >= 0 && id < p.V;
    t = have ? t : -INFINITY;
    s_id[k] = have ? (int)id : -1;
    s_p[k] = t;
    top = t != t ? t : fmaxf(top, t);
  }
  // NaN must survive the maximum: it is carried as the sum instead
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
  top = red[0][0];
#pragma unroll
  for (int w = 1; w < kDsWarps; ++w) top = fmaxf(top, red[0][w]);
  float mass = 0.f;
  for (int k = tid; k < p.K; k += kDsThreads) {
    if (top == -INFINITY) mass += s_p[k] == -INFINITY ? 0.f : s_p[k];  // no entry, or NaN
    else mass += ds_exp((s_p[k] - top) * inv_tau);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  if (lane == 0) red[1][warp] = mass;
  __syncthreads();
  mass = red[1][0];
#pragma unroll
  for (int w = 1; w < kDsWarps; ++w) mass += red[1][w];
  const bool empty = mass == 0.f;
  const float log_mass = logf(mass), inv_mass = 1.0f / mass;

  float lse = 0.f;
  if constexpr (kMode != kDsGrad) {
    MaxSum a{-INFINITY, 0.f};
    for (int s0 = begin + tid; s0 < end; s0 += 4 * kDsThreads) {
      uint4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (s0 + u * kDsThreads < end) w[u] = load(s0 + u * kDsThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int slot = s0 + u * kDsThreads;
        if (slot >= end) break;
        float v[N];
        slot_values<E>(w[u], v);
        const bool edge = slot * N < phase || (slot + 1) * N > p.V + phase;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_s(v[i]);
        if (kCap && edge) {  // tanh turned the places outside the row into -c
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int e = slot * N + i - phase;
            if (e < 0 || e >= p.V) v[i] = -INFINITY;
          }
        }
        if constexpr (kHold) {
          if constexpr (kCap) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
              reinterpret_cast<float4*>(hold)[i * share + slot - begin] =
                  make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          } else {
            hold[slot - begin] = w[u];
          }
        }
        float m = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
        if (m > a.m) {
          a.s = a.m == -INFINITY ? a.s : a.s * ds_exp(a.m - m);
          a.m = m;
        }
        const float base = a.m == -INFINITY ? 0.f : a.m;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += ds_exp(v[i] - base);
        a.s += sum;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, a.m, o), os = __shfl_xor_sync(0xffffffffu, a.s, o);
      a.join(om, os);
    }
    __syncthreads();  // red's earlier readers are done
    if (lane == 0) red[0][warp] = a.m, red[1][warp] = a.s;
    __syncthreads();
    a = MaxSum{red[0][0], red[1][0]};
#pragma unroll
    for (int w = 1; w < kDsWarps; ++w) a.join(red[0][w], red[1][w]);
    if (p.parts > 1) {
      if (tid == 0) part = make_float2(a.m, a.s);
      cluster_sync();
      MaxSum all{-INFINITY, 0.f};
      for (int r = 0; r < p.parts; ++r) {
        const uint32_t at = cluster_addr(&part, (uint32_t)r);
        all.join(__uint_as_float(ld_cluster_u32(at)), __uint_as_float(ld_cluster_u32(at + 4)));
      }
      a = all;
      cluster_sync();  // no CTA of the cluster leaves while another reads its part
    }
    lse = a.m == -INFINITY ? logf(a.s) : a.m + logf(a.s);
  } else {
    lse = __ldg(p.lse_in + row);
  }

  if (kMode != kDsGrad && rank == 0) {
    float l = 0.f;
    for (int k = tid; k < p.K; k += kDsThreads) {
      if (s_id[k] < 0) continue;
      const float t = (s_p[k] - top) * inv_tau, pk = ds_exp(t) * inv_mass;
      if (pk != 0.f) l += pk * ((t - log_mass) + (lse - to_s(to_f32(z[s_id[k]]))));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncthreads();
    if (lane == 0) red[0][warp] = l;
    __syncthreads();
    if (tid == 0) {
      l = red[0][0];
#pragma unroll
      for (int w = 1; w < kDsWarps; ++w) l += red[0][w];
      p.loss[row] = empty ? 0.f : p.tau * p.tau * l;
      if (p.lse) p.lse[row] = lse;
    }
  }

  if constexpr (kMode != kDsLoss) {
    E* g = reinterpret_cast<E*>(p.grad) + row * p.grad_ld;
    const bool same = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(E)) == phase;
    const float up = p.tau * (p.up ? __ldg(p.up + row) : 1.0f);
    const float th_of = kCap ? p.tau * inv_cap : 0.f;  // tanh(z / c) = s tau / c
    // gradient at a column whose entries hold the mass pj
    auto value = [&](float s, float pj) {
      float v = up * (ds_exp(s - lse) - pj);
      if (kCap) {
        const float th = s * th_of;
        v *= fmaf(-th, th, 1.0f);
      }
      return empty ? 0.f : v;
    };
    for (int slot = begin + tid; slot < end; slot += kDsThreads) {
      float v[N];
      if constexpr (kHold && kCap) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
          const float4 f = reinterpret_cast<const float4*>(hold)[i * share + slot - begin];
          v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
        }
      } else {
        slot_values<E>(kHold ? hold[slot - begin] : load(slot), v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_s(v[i]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = value(v[i], 0.f);
      if (same && slot * N >= phase && (slot + 1) * N <= p.V + phase) {
        __stcs(reinterpret_cast<uint4*>(g - phase) + slot, slot_pack<E>(v));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int e = slot * N + i - phase;
          if (e >= 0 && e < p.V) g[e] = from_f32<E>(v[i]);
        }
      }
    }
    if (empty) return;
    __syncthreads();  // the dense stores of this CTA come before its entries' stores
    const int e0 = begin * N - phase, e1 = min(p.V, end * N - phase);
    for (int k = tid; k < p.K; k += kDsThreads) {
      const int id = s_id[k];
      if (id < 0 || id < e0 || id >= e1) continue;
      bool first = true, again = false;
      for (int i = 0; i < p.K; ++i) {
        if (s_id[i] != id || i == k) continue;
        if (i < k) first = false;
        else again = true;
      }
      if (!first) continue;
      float pj = ds_exp((s_p[k] - top) * inv_tau) * inv_mass;
      if (again)
        for (int i = k + 1; i < p.K; ++i)
          if (s_id[i] == id) pj += ds_exp((s_p[i] - top) * inv_tau) * inv_mass;
      g[id] = from_f32<E>(value(to_s(to_f32(z[id])), pj));
    }
  }
}

int device_sm_count();

// Bytes of shared memory that `parts` CTAs each need to hold their part of a row.
static int64_t ds_hold_bytes(int V, int elem, bool cap, int parts) {
  const int n = 16 / elem;
  const int64_t slots = ((int64_t)V + 2 * n - 1) / n;
  const int64_t share = (slots + parts - 1) / parts;
  return share * (cap ? 4 * n : 16);
}

template <typename E, int kMode, bool kCap>
static int launch_distill(DistillParams& p, cudaStream_t s) {
  static KernelOptIn opt_in;
  // The fewest CTAs per row that give every SM two, of at least 1,024 slots (four loads a thread); more
  // where the row must fit shared memory.
  const int64_t slots = ((int64_t)p.V + DsSlot<E>::kN - 1) / DsSlot<E>::kN;
  const int64_t want = 2 * (int64_t)device_sm_count();
  int parts = 1;
  while (parts < kDsMaxCluster && p.rows * parts < want && slots / (2 * parts) >= kDsThreads) parts *= 2;
  int smem = 0;
  if (kMode == kDsBoth) {
    while (parts < kDsMaxCluster && ds_hold_bytes(p.V, sizeof(E), kCap, parts) > kDsRowBytes / 4) parts *= 2;
    const int64_t need = ds_hold_bytes(p.V, sizeof(E), kCap, parts);
    if (need > kDsRowBytes) return kStatusUnsupported;
    smem = (int)need;
  }
  if (p.rows * parts > INT32_MAX) return kStatusUnsupported;
  p.parts = parts;
  if (!opt_in(distill_kernel<E, kMode, kCap>, kMode == kDsBoth ? kDsRowBytes : 0)) return kStatusLaunchFailed;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)parts, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.rows * parts)), cfg.blockDim = dim3(kDsThreads);
  cfg.dynamicSmemBytes = (size_t)smem, cfg.stream = s;
  cfg.attrs = &attr, cfg.numAttrs = kMode == kDsGrad ? 0 : 1;  // the gradient's CTAs share nothing
  LaunchScope scope(kKindLoss, s);
  if (cudaLaunchKernelEx(&cfg, distill_kernel<E, kMode, kCap>, p) != cudaSuccess) {
    cudaGetLastError();
    return kStatusLaunchFailed;
  }
  return kStatusOk;
}

template <typename E>
static int launch_distill_mode(DistillParams& p, int mode, cudaStream_t s) {
  const bool cap = p.cap > 0.f;
  if (mode == kDsLoss) return cap ? launch_distill<E, kDsLoss, true>(p, s) : launch_distill<E, kDsLoss, false>(p, s);
  if (mode == kDsGrad) return cap ? launch_distill<E, kDsGrad, true>(p, s) : launch_distill<E, kDsGrad, false>(p, s);
  return cap ? launch_distill<E, kDsBoth, true>(p, s) : launch_distill<E, kDsBoth, false>(p, s);
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
