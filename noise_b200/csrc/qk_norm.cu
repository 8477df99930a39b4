// Norms of the queries and keys for each head with the position rotation, in one pass over both, and
// their gradients.
//
// A row is one head of one token, D values; (c, s) is the table's row at the token's position and
// R x = (x1 c + x2 s, -x1 s + x2 c) on the halves (x1, x2) of a row (utils/model.py:55-58).
//   rotate, then norm (utils/model.py:86-88):  u = R x,  y = w * u r,    r = (mean u^2 + eps)^(-1/2)
//   norm, then rotate:                         y = R (w * x r),          r = (mean x^2 + eps)^(-1/2)
// With z the norm's input, g the gradient of its output and n = z r:
//   dw = sum over the rows of g * n,   dz = r (h - n mean(n * h)),  h = g * w,
// and R's transpose (a, b) -> (a c - b s, a s + b c) carries a gradient back through the rotation.
//
// Bound: HBM. A pass reads and writes each value once (the gradient reads x and dy and writes dx; the
// norm's factor is recomputed from x, which costs nothing beside reading it). A row belongs to
// D / 16 lanes of one warp, each with eight values of either half, so a pair (x1, x2) never leaves its
// lane and the mean is a shuffle over at most 16 lanes. A lane takes several heads of one token at a
// time: their loads are in flight together and share the table's values. Query and key rows go to
// different CTAs of one launch, so that the weight gradients need one accumulator set a thread.
#include "operators.cuh"
#include "profile.cuh"
#include "ptx.cuh"

namespace noise {

struct QkSide {
  const void* x;   // [B, T, heads, D], strides xs
  const void* dy;  // gradient pass: [B, T, heads, D], strides ds
  void* y;         // y, or dx in the gradient pass, strides ys
  const float* w;  // [D] or null
  int64_t xs[3], ds[3], ys[3];
  int heads, chunks;  // chunks: groups of heads that one lane group takes at a time
  int64_t units;      // B * T * chunks
  int blocks;         // CTAs of the launch that work on this side
};

struct QkParams {
  QkSide side[2];
  const float* rope;  // [table][D] cos | sin
  const int* positions;
  int64_t pos_b;  // batch stride of positions (0: one row for all sequences)
  int64_t table;
  int T, D, lanes, rotate_first;
  float eps;
  float* partial;  // gradient pass with weights: [blocks of both sides][D]
};

// One row's values: eight of the first half, eight of the second.
struct Row16 {
  float a[8], b[8];
};

__device__ __forceinline__ void rotate(Row16& r, const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x1 = r.a[i], x2 = r.b[i];
    r.a[i] = fmaf(x1, c[i], x2 * s[i]);
    r.b[i] = fmaf(x2, c[i], -x1 * s[i]);
  }
}

__device__ __forceinline__ void rotate_back(Row16& r, const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x1 = r.a[i], x2 = r.b[i];
    r.a[i] = fmaf(x1, c[i], -x2 * s[i]);
    r.b[i] = fmaf(x1, s[i], x2 * c[i]);
  }
}

// Sum over the row's lane group (a power of two of lanes; the lanes past D / 16 hold zeros).
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float square_sum(const Row16& r) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = fmaf(r.a[i], r.a[i], fmaf(r.b[i], r.b[i], t));
  return t;
}

__device__ __forceinline__ float dot(const Row16& p, const Row16& q) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = fmaf(p.a[i], q.a[i], fmaf(p.b[i], q.b[i], t));
  return t;
}

constexpr int kQkThreads = 256;

// IT heads of a token per lane group and step.
template <typename E, int IT, bool kGrad>
__global__ void __launch_bounds__(kQkThreads) qk_norm_kernel(const __grid_constant__ QkParams p) {
  const bool key = (int)blockIdx.x >= p.side[0].blocks;
  const QkSide& S = p.side[key];
  const int block = key ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  const int lanes = p.lanes, half = p.D / 2;
  const int gl = threadIdx.x & (lanes - 1);          // lane of the row's group
  const int groups = kQkThreads / lanes, group = threadIdx.x / lanes;
  const bool on = gl * 16 < p.D;
  const int col = on ? gl * 8 : 0;
  const float inv_d = 1.0f / (float)p.D;
  float wa[8], wb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wa[i] = S.w ? __ldg(S.w + col + i) : 1.f;
    wb[i] = S.w ? __ldg(S.w + half + col + i) : 1.f;
  }
  Row16 dw;
  if (kGrad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) dw.a[i] = dw.b[i] = 0.f;
  }
  // Every lane runs the same number of steps: the shuffles below need the whole warp.
  for (int64_t u0 = (int64_t)block * groups; u0 < S.units; u0 += (int64_t)S.blocks * groups) {
    const int64_t unit = u0 + group;
    const bool live = on && unit < S.units;
    const int64_t token = live ? unit / S.chunks : 0;
    const int h0 = live ? (int)(unit - token * S.chunks) * IT : 0;
    const int64_t b = token / p.T, t = token - b * p.T;
    const E* x = reinterpret_cast<const E*>(S.x) + b * S.xs[0] + t * S.xs[1] + col;
    const E* dy = kGrad ? reinterpret_cast<const E*>(S.dy) + b * S.ds[0] + t * S.ds[1] + col : nullptr;
    Vec8<E> va[IT], vb[IT], ga[kGrad ? IT : 1], gb[kGrad ? IT : 1];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const bool have = live && h0 + i < S.heads;
      va[i].zero(), vb[i].zero();
      if (have) va[i].load(x + (h0 + i) * S.xs[2]), vb[i].load(x + (h0 + i) * S.xs[2] + half);
      if constexpr (kGrad) {
        ga[i].zero(), gb[i].zero();
        if (have) ga[i].load(dy + (h0 + i) * S.ds[2]), gb[i].load(dy + (h0 + i) * S.ds[2] + half);
      }
    }
    const int64_t pos = p.positions ? (int64_t)__ldg(p.positions + b * p.pos_b + t) : t;
    float c[8], s[8];
    // a position outside the table has no rotation: its rows come out as NaN
    const bool known = pos >= 0 && pos < p.table;
    if (known) {
      Vec8<float> tc, ts;
      tc.load(p.rope + pos * p.D + col), ts.load(p.rope + pos * p.D + half + col);
      tc.get(c), ts.get(s);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
    E* y = reinterpret_cast<E*>(S.y) + b * S.ys[0] + t * S.ys[1] + col;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      Row16 z;
      va[i].get(z.a), vb[i].get(z.b);
      if (p.rotate_first) rotate(z, c, s);
      if (!on) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z.a[j] = z.b[j] = 0.f;  // lanes without columns add nothing (not NaN)
      }
      const float r = rsqrtf(fmaf(group_sum(square_sum(z), lanes), inv_d, p.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) z.a[j] *= r, z.b[j] *= r;
      if constexpr (!kGrad) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z.a[j] *= wa[j], z.b[j] *= wb[j];
        if (!p.rotate_first) rotate(z, c, s);
      } else {
        Row16 g;
        ga[i].get(g.a), gb[i].get(g.b);
        if (!p.rotate_first) rotate_back(g, c, s);
        if (!on) {
#pragma unroll
          for (int j = 0; j < 8; ++j) g.a[j] = g.b[j] = 0.f;
        }
        if (live && h0 + i < S.heads) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            dw.a[j] = fmaf(g.a[j], z.a[j], dw.a[j]);
            dw.b[j] = fmaf(g.b[j], z.b[j], dw.b[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) g.a[j] *= wa[j], g.b[j] *= wb[j];
        const float m = group_sum(dot(z, g), lanes) * inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) z.a[j] = r * (g.a[j] - z.a[j] * m), z.b[j] = r * (g.b[j] - z.b[j] * m);
        if (p.rotate_first) rotate_back(z, c, s);
      }
      if (live && h0 + i < S.heads) {
        Vec8<E> o;
        o.set(z.a), o.store(y + (h0 + i) * S.ys[2]);
        o.set(z.b), o.store(y + (h0 + i) * S.ys[2] + half);
      }
    }
  }
  if constexpr (kGrad) {
    if (!S.w) return;
    // the CTA's sum: lanes of the same columns within a warp, then the warps in order
    __shared__ float part[kQkThreads / 32][256];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      for (int o = 16; o >= lanes; o >>= 1) {
        dw.a[i] += __shfl_xor_sync(0xffffffffu, dw.a[i], o);
        dw.b[i] += __shfl_xor_sync(0xffffffffu, dw.b[i], o);
      }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane < lanes && on) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[warp][col + i] = dw.a[i], part[warp][half + col + i] = dw.b[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += kQkThreads) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kQkThreads / 32; ++k) t += part[k][i];
      p.partial[(int64_t)blockIdx.x * p.D + i] = t;
    }
  }
}

// dw[i] = the sum over one side's CTAs of partial[block][i]: 32 columns a CTA, the blocks dealt to 32
// warps and their sums added in order, so that the result does not depend on the launch's timing.
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float* __restrict__ partial, int blocks_q,
                                                             int blocks_k, int D, float* __restrict__ dwq,
                                                             float* __restrict__ dwk) {
  __shared__ float part[32][33];
  float* out = blockIdx.y ? dwk : dwq;
  if (!out) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const int first = blockIdx.y ? blocks_q : 0, n = blockIdx.y ? blocks_k : blocks_q;
  float t = 0.f;
  if (col < D)
    for (int i = warp; i < n; i += 32) t += partial[(int64_t)(first + i) * D + col];
  part[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && col < D) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += part[i][lane];
    out[col] = t;
  }
}

int device_sm_count();

// CTAs of a gradient pass: at most this many per SM in all, so that the weight sums stay short.
constexpr int kQkGradBlocksPerSm = 8;
constexpr int kQkMaxBlocks = 4096;

// Splits one side's units over CTAs: one step each, or an even share of `cap` CTAs.
static void qk_side(QkSide& s, int64_t tokens, int it, int lanes, int64_t cap) {
  s.chunks = (s.heads + it - 1) / it;
  s.units = tokens * s.chunks;
  const int64_t groups = kQkThreads / lanes;
  int64_t blocks = (s.units + groups - 1) / groups;
  if (blocks > cap) blocks = cap;
  s.blocks = (int)(blocks < 1 ? 1 : blocks);
}

template <typename E, int IT, bool kGrad>
static void launch_qk(const QkParams& p, cudaStream_t s) {
  qk_norm_kernel<E, IT, kGrad><<<p.side[0].blocks + p.side[1].blocks, kQkThreads, 0, s>>>(p);
}

static bool qk_tensor_ok(const void* ptr, const int64_t* stride, int elem) {
  if (!ptr || !is_aligned(ptr, 16)) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] * elem % 16) return false;
  return true;
}

}  // namespace noise

using namespace noise;

extern "C" int64_t noise_qk_norm_workspace_bytes(int D) {
  return D < 16 || D > 256 ? -1 : (int64_t)2 * kQkMaxBlocks * D * 4;
}

extern "C" int noise_qk_norm_rope(const NoiseQkNorm* a, int backward, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (!a || !a->rope || a->B < 0 || a->T < 0 || a->H < 1 || a->Hk < 1 || a->table < 1) return kStatusBadArgument;
  if (a->D < 16 || a->D > 256 || a->D % 16) return kStatusUnsupported;
  if (a->dtype != NOISE_FP32 && a->dtype != NOISE_BF16 && a->dtype != NOISE_FP16) return kStatusUnsupported;
  if (a->B == 0 || a->T == 0) {  // no rows: the weights' gradients are zero
    cudaStream_t s0 = reinterpret_cast<cudaStream_t>(stream);
    for (float* g : {a->dwq, a->dwk})
      if (backward && g && cudaMemsetAsync(g, 0, a->D * 4, s0) != cudaSuccess) return kStatusLaunchFailed;
    return kStatusOk;
  }
  const int elem = a->dtype == NOISE_FP32 ? 4 : 2;
  if (!is_aligned(a->rope, 16)) return kStatusBadArgument;
  if (!qk_tensor_ok(a->q, a->q_stride, elem) || !qk_tensor_ok(a->k, a->k_stride, elem) ||
      !qk_tensor_ok(a->q_out, a->q_out_stride, elem) || !qk_tensor_ok(a->k_out, a->k_out_stride, elem))
    return kStatusBadArgument;
  if (backward && (!qk_tensor_ok(a->dq, a->dq_stride, elem) || !qk_tensor_ok(a->dk, a->dk_stride, elem)))
    return kStatusBadArgument;
  const bool weights = backward && (a->wq || a->wk);
  if (backward && ((a->wq != nullptr) != (a->dwq != nullptr) || (a->wk != nullptr) != (a->dwk != nullptr)))
    return kStatusBadArgument;
  if (weights && (!workspace || workspace_bytes < (size_t)noise_qk_norm_workspace_bytes(a->D)))
    return kStatusWorkspaceTooSmall;
  QkParams p{};
  p.side[0].x = a->q, p.side[0].dy = a->dq, p.side[0].y = a->q_out, p.side[0].w = a->wq, p.side[0].heads = a->H;
  p.side[1].x = a->k, p.side[1].dy = a->dk, p.side[1].y = a->k_out, p.side[1].w = a->wk, p.side[1].heads = a->Hk;
  for (int i = 0; i < 3; ++i) {
    p.side[0].xs[i] = a->q_stride[i], p.side[0].ds[i] = a->dq_stride[i], p.side[0].ys[i] = a->q_out_stride[i];
    p.side[1].xs[i] = a->k_stride[i], p.side[1].ds[i] = a->dk_stride[i], p.side[1].ys[i] = a->k_out_stride[i];
  }
  p.rope = a->rope, p.positions = a->positions, p.pos_b = a->positions_stride, p.table = a->table;
  p.T = a->T, p.D = a->D, p.rotate_first = a->order == NOISE_ROTATE_NORM, p.eps = a->eps;
  p.lanes = 1;
  while (p.lanes * 16 < a->D) p.lanes *= 2;
  p.partial = reinterpret_cast<float*>(workspace);
  const int64_t tokens = (int64_t)a->B * a->T;
  const bool wide = a->dtype == NOISE_FP32;
  const int it = backward ? (wide ? 1 : 2) : (wide ? 2 : 4);
  int64_t cap = INT32_MAX / 2;
  if (weights) cap = min((int64_t)kQkMaxBlocks, (int64_t)device_sm_count() * kQkGradBlocksPerSm);
  qk_side(p.side[0], tokens, it, p.lanes, cap);
  qk_side(p.side[1], tokens, it, p.lanes, cap);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  LaunchScope scope(kKindOther, s, weights ? 2 : 1);
  if (!backward) {
    if (a->dtype == NOISE_FP32) launch_qk<float, 2, false>(p, s);
    else if (a->dtype == NOISE_BF16) launch_qk<__nv_bfloat16, 4, false>(p, s);
    else launch_qk<__half, 4, false>(p, s);
  } else {
    if (a->dtype == NOISE_FP32) launch_qk<float, 1, true>(p, s);
    else if (a->dtype == NOISE_BF16) launch_qk<__nv_bfloat16, 2, true>(p, s);
    else launch_qk<__half, 2, true>(p, s);
    if (weights)
      qk_weight_sum_kernel<<<dim3((a->D + 31) / 32, 2), 1024, 0, s>>>(p.partial, p.side[0].blocks, p.side[1].blocks, a->D,
                                                                      a->dwq, a->dwk);
  }
  return cudaGetLastError() == cudaSuccess ? kStatusOk : kStatusLaunchFailed;
}
