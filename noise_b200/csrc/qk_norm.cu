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
// D / 8 lanes of one warp, each with four values of either half, so a pair (x1, x2) never leaves its
// lane and the mean is a shuffle over the row's lanes. A lane takes several heads of one token at a
// time: their loads are in flight together and share the table's values. Query and key rows go to
// different CTAs of one launch, so that the weight gradients need one accumulator set a thread.
//
// Measured: 8 + 8 heads of 64 in 16,384 tokens of a packed bf16 projection: 16.4 us, 4.1 TB/s. 12 + 4 heads of 96 in
// 22,662 tokens with weights: forward 37 us, 3.7 TB/s, gradient 63 us with the weights' sums, 3.3 TB/s; in fp32 50 and 79
// us, 5.5 and 5.3 TB/s. Next to HBM stand the instructions (120 a lane and row forward, 206 in the gradient; 60 % of the
// issue slots) and their latency at 32 warps an SM. A row takes a power of two of lanes, so that a quarter of them have no
// columns at D = 96 and three eighths at 80: they take issue slots all the same. Eight values of either half a lane save instructions and cost registers: 97 against 60 us for
// the gradient; copies through a ring in shared memory, 68 against 58; arithmetic without pairs, 24 instructions more,
// the same time.
#include <algorithm>
#include <utility>

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
  int heads;
  FastDiv chunks;  // groups of heads that one lane group takes at a time
  uint32_t units;  // B * T * chunks
  int blocks;      // CTAs of the launch that work on this side
};

struct QkParams {
  QkSide side[2];
  const float* rope;  // [table][D] cos | sin
  const int* positions;
  int64_t pos_b;  // batch stride of positions (0: one row for all sequences)
  int64_t table;
  FastDiv T;
  int D;
  float eps;
  float* partial;  // gradient pass with weights: [blocks of both sides][D]
};

// A lane's values of one row: four of the first half, four of the second, in pairs (the sm_100 f32x2 arithmetic).
struct RowPart {
  float2 a[2], b[2];
};

// R with ns = -s; its transpose with s and ns exchanged.
__device__ __forceinline__ void rotate(RowPart& r, const float2 (&c)[2], const float2 (&s)[2], const float2 (&ns)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 x1 = r.a[i], x2 = r.b[i];
    r.a[i] = __ffma2_rn(x1, c[i], __fmul2_rn(x2, s[i]));
    r.b[i] = __ffma2_rn(x2, c[i], __fmul2_rn(x1, ns[i]));
  }
}

// Sum over those of the row's lane group (a power of two of lanes) that are on: the ones below D / 8.
template <int kLanes>
__device__ __forceinline__ float group_sum(float2 t, bool on) {
  float v = on ? t.x + t.y : 0.f;
#pragma unroll
  for (int o = kLanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float2 dot(const RowPart& p, const RowPart& q) {
  float2 t = __fmul2_rn(p.a[0], q.a[0]);
  t = __ffma2_rn(p.a[1], q.a[1], t);
  t = __ffma2_rn(p.b[0], q.b[0], t);
  return __ffma2_rn(p.b[1], q.b[1], t);
}

__device__ __forceinline__ void scale_by(RowPart& r, const float2 (&a)[2], const float2 (&b)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) r.a[i] = __fmul2_rn(r.a[i], a[i]), r.b[i] = __fmul2_rn(r.b[i], b[i]);
}

constexpr int kQkThreads = 256;

// IT heads of a token per lane group and step.
template <typename E, int IT, bool kGrad, bool kRotateFirst, int kLanes>
__global__ void __launch_bounds__(kQkThreads, 4) qk_norm_kernel(const __grid_constant__ QkParams p) {
  const bool key = (int)blockIdx.x >= p.side[0].blocks;
  const QkSide& S = p.side[key];
  const int block = key ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  constexpr int lanes = kLanes;
  const int half = p.D / 2;
  const int gl = threadIdx.x & (lanes - 1);          // lane of the row's group
  const int groups = kQkThreads / lanes, group = threadIdx.x / lanes;
  const bool on = gl * 8 < p.D;
  const int col = on ? gl * 4 : 0;
  const float inv_d = 1.0f / (float)p.D;
  float2 wa[2], wb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    wa[i] = S.w ? make_float2(__ldg(S.w + col + 2 * i), __ldg(S.w + col + 2 * i + 1)) : make_float2(1.f, 1.f);
    wb[i] = S.w ? make_float2(__ldg(S.w + half + col + 2 * i), __ldg(S.w + half + col + 2 * i + 1)) : make_float2(1.f, 1.f);
  }
  RowPart dw;
  if (kGrad) {
#pragma unroll
    for (int i = 0; i < 2; ++i) dw.a[i] = dw.b[i] = make_float2(0.f, 0.f);
  }
  // Every lane runs the same number of steps: the shuffles below need the whole warp.
  for (uint32_t u0 = (uint32_t)block * groups; u0 < S.units; u0 += (uint32_t)S.blocks * groups) {
    // Lanes without columns and groups without a unit load what others load too (unit 0, columns 0): nothing but
    // their sums and stores has to be held back. So do rows behind the last head of a token.
    const bool live = u0 + group < S.units;
    const uint32_t unit = live ? u0 + group : 0;
    const uint32_t token = S.chunks(unit), h0 = (unit - token * S.chunks.d) * IT;
    const uint32_t b = p.T(token), t = token - b * p.T.d;
    const int heads = live && on ? S.heads - (int)h0 : 0;  // rows this lane works for
    const E* x = reinterpret_cast<const E*>(S.x) + b * S.xs[0] + t * S.xs[1] + h0 * S.xs[2] + col;
    const E* dy = kGrad ? reinterpret_cast<const E*>(S.dy) + b * S.ds[0] + t * S.ds[1] + h0 * S.ds[2] + col : nullptr;
    Vec4<E> va[IT], vb[IT], ga[kGrad ? IT : 1], gb[kGrad ? IT : 1];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      va[i].load(x), vb[i].load(x + half);
      if constexpr (kGrad) ga[i].load(dy), gb[i].load(dy + half);
      if (i + 1 < S.heads - (int)h0) {
        x += S.xs[2];
        if constexpr (kGrad) dy += S.ds[2];
      }
    }
    const int64_t pos = p.positions ? (int64_t)__ldg(p.positions + b * p.pos_b + t) : t;
    float2 c[2], s[2], ns[2];
    // a position outside the table has no rotation: its rows come out as NaN
    if (pos >= 0 && pos < p.table) {
      const float4 tc = __ldg(reinterpret_cast<const float4*>(p.rope + pos * p.D + col));
      const float4 ts = __ldg(reinterpret_cast<const float4*>(p.rope + pos * p.D + half + col));
      c[0] = make_float2(tc.x, tc.y), c[1] = make_float2(tc.z, tc.w);
      s[0] = make_float2(ts.x, ts.y), s[1] = make_float2(ts.z, ts.w);
    } else {
      c[0] = c[1] = s[0] = s[1] = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) ns[i] = make_float2(-s[i].x, -s[i].y);
    E* y = reinterpret_cast<E*>(S.y) + b * S.ys[0] + t * S.ys[1] + h0 * S.ys[2] + col;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      RowPart z;
      va[i].get(z.a), vb[i].get(z.b);
      if (kRotateFirst) rotate(z, c, s, ns);
      const float r = rsqrtf(fmaf(group_sum<kLanes>(dot(z, z), on), inv_d, p.eps));
      const float2 r2[2] = {make_float2(r, r), make_float2(r, r)};
      scale_by(z, r2, r2);
      if constexpr (!kGrad) {
        if (S.w) scale_by(z, wa, wb);
        if (!kRotateFirst) rotate(z, c, s, ns);
      } else {
        RowPart g;
        ga[i].get(g.a), gb[i].get(g.b);
        if (!kRotateFirst) rotate(g, c, ns, s);
        if (S.w) {
          if (i < heads) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              dw.a[j] = __ffma2_rn(g.a[j], z.a[j], dw.a[j]), dw.b[j] = __ffma2_rn(g.b[j], z.b[j], dw.b[j]);
          }
          scale_by(g, wa, wb);
        }
        const float m = group_sum<kLanes>(dot(z, g), on) * -inv_d;
        const float2 m2 = make_float2(m, m);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          z.a[j] = __fmul2_rn(__ffma2_rn(z.a[j], m2, g.a[j]), r2[0]);
          z.b[j] = __fmul2_rn(__ffma2_rn(z.b[j], m2, g.b[j]), r2[0]);
        }
        if (kRotateFirst) rotate(z, c, ns, s);
      }
      if (i < heads) {
        Vec4<E> o;
        o.set(z.a), o.store(y);
        o.set(z.b), o.store(y + half);
        y += S.ys[2];
      }
    }
  }
  if constexpr (kGrad) {
    if (!S.w) return;
    // the CTA's sum: lanes of the same columns within a warp, then the warps in order
    __shared__ float part[kQkThreads / 32][256];
    float sum[8] = {dw.a[0].x, dw.a[0].y, dw.a[1].x, dw.a[1].y, dw.b[0].x, dw.b[0].y, dw.b[1].x, dw.b[1].y};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int o = 16; o >= lanes; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane < lanes && on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][col + i] = sum[i], part[warp][half + col + i] = sum[4 + i];
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
#pragma unroll 8
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

// A gradient pass with weights runs in one wave of CTAs, dealt to the two sides by their work, so that there are
// few sums of weight gradients to add up.
constexpr int kQkBlocksPerSm = 4;
constexpr int kQkMaxBlocks = 4096;  // of both sides

// Splits one side's units over CTAs: one step each, or an even share of `cap` CTAs.
static bool qk_side(QkSide& s, int64_t tokens, int it, int lanes, int64_t cap) {
  const int64_t chunks = (s.heads + it - 1) / it, units = tokens * chunks, groups = kQkThreads / lanes;
  const int64_t blocks = min((units + groups - 1) / groups, cap);
  if (units + blocks * groups > INT32_MAX) return false;  // unit numbers and their steps stay below 2^31
  s.chunks = FastDiv((uint32_t)chunks), s.units = (uint32_t)units, s.blocks = (int)blocks;
  return true;
}

template <typename E, int IT, bool kGrad, bool kRotateFirst>
static void launch_qk(const QkParams& p, int lanes, cudaStream_t s) {
  const int blocks = p.side[0].blocks + p.side[1].blocks;
  switch (lanes) {
    case 2: return qk_norm_kernel<E, IT, kGrad, kRotateFirst, 2><<<blocks, kQkThreads, 0, s>>>(p);
    case 4: return qk_norm_kernel<E, IT, kGrad, kRotateFirst, 4><<<blocks, kQkThreads, 0, s>>>(p);
    case 8: return qk_norm_kernel<E, IT, kGrad, kRotateFirst, 8><<<blocks, kQkThreads, 0, s>>>(p);
    case 16: return qk_norm_kernel<E, IT, kGrad, kRotateFirst, 16><<<blocks, kQkThreads, 0, s>>>(p);
    default: return qk_norm_kernel<E, IT, kGrad, kRotateFirst, 32><<<blocks, kQkThreads, 0, s>>>(p);
  }
}

template <typename E, int IT, bool kGrad>
static void launch_qk(const QkParams& p, bool rotate_first, int lanes, cudaStream_t s) {
  rotate_first ? launch_qk<E, IT, kGrad, true>(p, lanes, s) : launch_qk<E, IT, kGrad, false>(p, lanes, s);
}

static bool qk_tensor_ok(const void* ptr, const int64_t* stride, int elem) {
  if (!ptr || !is_aligned(ptr, 16)) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] * elem % 16) return false;
  return true;
}

// Rows of `bytes` bytes at p + stride . i, 0 <= i < n.
struct QkRows {
  int64_t p, n[3], stride[3], bytes;
  QkRows(const void* ptr, int B, int T, int heads, const int64_t* st, int D, int elem)
      : p((int64_t)reinterpret_cast<uintptr_t>(ptr)), n{B, T, heads}, stride{st[0] * elem, st[1] * elem, st[2] * elem},
        bytes((int64_t)D * elem) {}
  bool same(const QkRows& o) const {  // the same rows in the same places
    bool all = p == o.p;
    for (int i = 0; i < 3; ++i) all = all && n[i] == o.n[i] && (n[i] == 1 || stride[i] == o.stride[i]);
    return all;
  }
  bool within(int64_t begin, int64_t end) const {  // its extent reaches into [begin, end)
    int64_t lo = p, hi = p + bytes;
    for (int i = 0; i < 3; ++i) (stride[i] < 0 ? lo : hi) += (n[i] - 1) * stride[i];
    return lo < end && begin < hi;
  }
};

// Whether two rows meet: integers x_k in [lo_k, hi_k] with |d + sum_k step_k x_k| < bytes, and, of one set of rows against
// itself, not all 0. The widest step first, each within what the narrower ones can still make up: two or three values a
// step where rows are nested as in any view of a tensor. A search that gets long is taken for an overlap.
struct QkMeet {
  struct Step {
    int64_t step, lo, hi;
  } s[6];
  int n = 0, budget = 1 << 14;
  int64_t bytes;
  bool self;

  void add(int64_t step, int64_t lo, int64_t hi) {
    if (step < 0) step = -step, std::swap(lo, hi), lo = -lo, hi = -hi;
    if (!step && !self) return;  // the same rows again
    for (int i = 0; i < n && !self; ++i)
      if (s[i].step == step) {
        s[i].lo += lo, s[i].hi += hi;
        return;
      }
    s[n++] = {step, lo, hi};
  }
  bool search(int k, int64_t d, bool zero) {
    if (--budget < 0) return true;
    if (k == n) return d > -bytes && d < bytes && !(self && zero);
    int64_t lo = d - bytes + 1, hi = d + bytes - 1;  // what this step has to bring to 0
    for (int i = k + 1; i < n; ++i) lo += s[i].step * s[i].lo, hi += s[i].step * s[i].hi;
    int64_t first = s[k].lo, last = s[k].hi;
    if (s[k].step) {  // step x in [-hi, -lo], rounded inwards
      auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
      first = std::max(first, -floor_div(hi, s[k].step)), last = std::min(last, floor_div(-lo, s[k].step));
    }
    for (int64_t x = first; x <= last; ++x)
      if (search(k + 1, d + s[k].step * x, zero && x == 0)) return true;
    return false;
  }
  static bool run(const QkRows& a, const QkRows& b, bool self) {
    QkMeet m;
    m.bytes = a.bytes, m.self = self;
    for (int i = 0; i < 3; ++i) {
      if (!a.n[i] || !b.n[i]) return false;
      if (self) {
        if (a.n[i] > 1) m.add(a.stride[i], -(a.n[i] - 1), a.n[i] - 1);
        continue;
      }
      m.add(a.stride[i], 0, a.n[i] - 1);
      m.add(-b.stride[i], 0, b.n[i] - 1);
    }
    std::sort(m.s, m.s + m.n, [](const Step& x, const Step& y) { return x.step > y.step; });
    return m.search(0, a.p - b.p, true);
  }
};

static bool qk_overlap(const NoiseQkNorm* a, bool backward) {
  if (a->B < 1 || a->T < 1 || a->H < 1 || a->Hk < 1) return false;
  const int elem = a->dtype == NOISE_FP32 ? 4 : 2;
  auto rows = [&](const void* p, int heads, const int64_t* st) { return QkRows(p, a->B, a->T, heads, st, a->D, elem); };
  const QkRows out[2] = {rows(a->q_out, a->H, a->q_out_stride), rows(a->k_out, a->Hk, a->k_out_stride)};
  const QkRows in[4] = {rows(a->q, a->H, a->q_stride), rows(a->k, a->Hk, a->k_stride), rows(a->dq, a->H, a->dq_stride),
                        rows(a->dk, a->Hk, a->dk_stride)};
  auto apart = [](const QkRows& x, const QkRows& y) {
    int64_t lo = y.p, hi = y.p + y.bytes;
    for (int i = 0; i < 3; ++i) (y.stride[i] < 0 ? lo : hi) += (y.n[i] - 1) * y.stride[i];
    return !x.within(lo, hi) || !QkMeet::run(x, y, false);
  };
  if (!apart(out[0], out[1])) return true;
  for (int o = 0; o < 2; ++o) {
    if (QkMeet::run(out[o], out[o], true)) return true;
    for (int i = 0; i < (backward ? 4 : 2); ++i)  // a thread reads its rows before it writes them: in place is fine
      if (!((i & 1) == o && out[o].same(in[i])) && !apart(out[o], in[i])) return true;
    auto reads = [&](const void* p, int64_t bytes) {
      const int64_t at = (int64_t)reinterpret_cast<uintptr_t>(p);
      return p && out[o].within(at, at + bytes);
    };
    if (reads(a->rope, a->table * a->D * 4) || reads(a->wq, a->D * 4) || reads(a->wk, a->D * 4) ||
        reads(a->positions, ((a->B - 1) * a->positions_stride + a->T) * 4))
      return true;
  }
  return false;
}

}  // namespace noise

using namespace noise;

extern "C" int noise_qk_norm_overlap(const NoiseQkNorm* a, int backward) { return a && qk_overlap(a, backward != 0); }

extern "C" int64_t noise_qk_norm_workspace_bytes(int D) {
  return D < 16 || D > 256 ? -1 : (int64_t)kQkMaxBlocks * D * 4;
}

extern "C" int noise_qk_norm_rope(const NoiseQkNorm* a, int backward, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (!a || !a->rope || a->B < 0 || a->T < 0 || a->H < 1 || a->Hk < 1 || a->table < 1) return kStatusBadArgument;
  if (a->order != NOISE_ROTATE_NORM && a->order != NOISE_NORM_ROTATE) return kStatusBadArgument;
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
  if (qk_overlap(a, backward != 0)) return kStatusBadArgument;
  QkParams p{};
  p.side[0].x = a->q, p.side[0].dy = a->dq, p.side[0].y = a->q_out, p.side[0].w = a->wq, p.side[0].heads = a->H;
  p.side[1].x = a->k, p.side[1].dy = a->dk, p.side[1].y = a->k_out, p.side[1].w = a->wk, p.side[1].heads = a->Hk;
  for (int i = 0; i < 3; ++i) {
    p.side[0].xs[i] = a->q_stride[i], p.side[0].ds[i] = a->dq_stride[i], p.side[0].ys[i] = a->q_out_stride[i];
    p.side[1].xs[i] = a->k_stride[i], p.side[1].ds[i] = a->dk_stride[i], p.side[1].ys[i] = a->k_out_stride[i];
  }
  p.rope = a->rope, p.positions = a->positions, p.pos_b = a->positions_stride, p.table = a->table;
  p.T = FastDiv((uint32_t)a->T), p.D = a->D, p.eps = a->eps;
  int lanes = 2;
  while (lanes * 8 < a->D) lanes *= 2;
  p.partial = reinterpret_cast<float*>(workspace);
  const int64_t tokens = (int64_t)a->B * a->T;
  const bool wide = a->dtype == NOISE_FP32;
  const int it = backward ? (wide ? 1 : 2) : (wide ? 2 : 4);
  // The forward and a gradient without weights take one step a CTA.
  int64_t cap_q = INT32_MAX, cap_k = INT32_MAX;
  if (weights) {
    const int64_t all = min(kQkMaxBlocks, device_sm_count() * kQkBlocksPerSm);
    const int64_t q = (a->H + it - 1) / it, k = (a->Hk + it - 1) / it;
    cap_k = max((int64_t)1, all * k / (q + k)), cap_q = all - cap_k;
  }
  if (!qk_side(p.side[0], tokens, it, lanes, cap_q) || !qk_side(p.side[1], tokens, it, lanes, cap_k))
    return kStatusUnsupported;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  LaunchScope scope(kKindOther, s, weights ? 2 : 1);
  if (!backward) {
    if (a->dtype == NOISE_FP32) launch_qk<float, 2, false>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
    else if (a->dtype == NOISE_BF16) launch_qk<__nv_bfloat16, 4, false>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
    else launch_qk<__half, 4, false>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
  } else {
    if (a->dtype == NOISE_FP32) launch_qk<float, 1, true>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
    else if (a->dtype == NOISE_BF16) launch_qk<__nv_bfloat16, 2, true>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
    else launch_qk<__half, 2, true>(p, a->order == NOISE_ROTATE_NORM, lanes, s);
    if (weights)
      qk_weight_sum_kernel<<<dim3((a->D + 31) / 32, 2), 1024, 0, s>>>(p.partial, p.side[0].blocks, p.side[1].blocks, a->D,
                                                                      a->dwq, a->dwk);
  }
  return cudaGetLastError() == cudaSuccess ? kStatusOk : kStatusLaunchFailed;
}
