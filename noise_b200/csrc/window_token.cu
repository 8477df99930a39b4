// The single-token form of the sliding-window attention with sinks: one query per sequence and head over a
// cache, where only the visible keys (the sinks and the window's) are ever touched.
//
//   s_i = scale q . k_i over the visible keys,  out = sum_i exp(s_i) v_i / sum_i exp(s_i),  lse = log sum exp(s)
//
// Bound: HBM for many sequences (each visible key and value is read once), latency for a few. The heads
// that share a key head are the rows of one 16-row tile, so a key is read once for all of them. One CTA
// cluster works on one (sequence, key head): the keys are dealt to its CTAs and warps in chunks, each warp
// keeps its own running maximum, sum and output rows over its chunks (copied three stages ahead with
// cp.async), the warps of a CTA meet in shared memory and the CTAs of the cluster through distributed shared
// memory. One launch, no workspace, and the parts are joined in a fixed order.
// The products run on mma.sync m16n8k16 with fp32 accumulators: a tile of at most 16 query rows leaves a
// 128-row tensor-memory product mostly empty, and the bytes of the cache bound this form, not its products.
// Keys behind the sequence's end are not loaded (their places read as zeros), so a cache may hold anything there.
// Measured: 64 sequences over 8 K tokens of cache or fewer, 32 heads on 8 of 128: 175 us a call, 5.9 TB/s; one sequence,
// 8 heads of 64, 1,024 visible keys: 11.5 us a call, which is the host's time for it.
#include <atomic>
#include <type_traits>

#include "profile.cuh"
#include "window.cuh"

namespace noise {

template <int DP>
struct WinTok {
  static constexpr int kWarps = 4, kThreads = kWarps * 32;
  static constexpr int KC = DP == 64 ? 32 : 16;  // keys of a chunk
  static constexpr int kStages = 3;
  static constexpr int kPitch = DP * 2 + 16;     // a key's row in shared memory: 16 bytes of padding spread the banks
  static constexpr int kTile = KC * kPitch;
  static constexpr int kWarpBytes = kStages * 2 * kTile;
  static constexpr int kSmem = kWarps * kWarpBytes;
  // after the keys: each warp's O rows, then the CTA's
  static constexpr int kRowFloats = DP + 4;
  static_assert((kWarps + 1) * 16 * kRowFloats * 4 <= kSmem, "the partial outputs reuse the key stages");
};

struct TokenParams {
  const void *q, *k, *v;
  int64_t q_b, q_h, k_b, k_t, k_h, v_b, v_t, v_h;
  const int* lengths;
  void* out;
  float* lse;
  int H, group, tiles, Tk, D, window, sinks;
  float scale;
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename E>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<E, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) { return __uint_as_float(ld_cluster_u32(addr)); }

template <typename E, int DP, int kMost>  // at most kMost CTAs a cluster
__global__ void __launch_bounds__(WinTok<DP>::kThreads) window_token_kernel(const __grid_constant__ TokenParams p) {
  using L = WinTok<DP>;
  constexpr int KC = L::KC;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int parts = gridDim.x, rank = blockIdx.x;  // the cluster spans grid.x
  const int kv = blockIdx.y / p.tiles, first = (blockIdx.y - kv * p.tiles) * 16;  // first head row of this tile
  const int heads = min(16, p.group - first), b = blockIdx.z;
  const int head0 = kv * p.group + first;
  const int length = min(max(__ldg(p.lengths + b), 0), p.Tk);
  const int lo = max(0, length - 1 - p.window), ns = min(p.sinks, lo);
  const int n = length - lo + ns;  // visible keys: the sinks before the window, then the window
  const E* kb = reinterpret_cast<const E*>(p.k) + b * p.k_b + kv * p.k_h;
  const E* vb = reinterpret_cast<const E*>(p.v) + b * p.v_b + kv * p.v_h;

  // query rows as the products' A fragments, scaled by nothing: the scale is applied to the fp32 scores
  uint32_t qa[DP / 16][4];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = lane / 4 + (u & 1) * 8, col = 16 * s + (lane & 3) * 2 + (u >> 1) * 8;
      qa[s][u] = 0u;
      if (r < heads && col < p.D)
        qa[s][u] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const E*>(p.q) + b * p.q_b + (head0 + r) * p.q_h + col);
    }

  const uint32_t stage0 = smem_u32(smem) + warp * L::kWarpBytes;
  const int chunks = (n + KC - 1) / KC, step = parts * L::kWarps, mine = rank * L::kWarps + warp;
  auto fetch = [&](int c, int stage) {  // chunk c of the sequence into a stage of this warp
    const uint32_t ks = stage0 + stage * 2 * L::kTile, vs = ks + L::kTile;
#pragma unroll
    for (int e = lane; e < KC * (DP / 8); e += 32) {
      const int row = e / (DP / 8), col = (e % (DP / 8)) * 8, i = c * KC + row;
      const bool have = i < n && col < p.D;
      const int64_t key = have ? (i < ns ? i : lo + i - ns) : 0;
      const int at = have ? col : 0;
      cp_async16(ks + row * L::kPitch + col * 2, kb + key * p.k_t + at, have);
      cp_async16(vs + row * L::kPitch + col * 2, vb + key * p.v_t + at, have);
    }
  };
  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows lane / 4 and lane / 4 + 8
  const float c2 = p.scale * 1.4426950408889634f;
#pragma unroll
  for (int s = 0; s < L::kStages - 1; ++s) {
    if (mine + s * step < chunks) fetch(mine + s * step, s);
    cp_async_commit();
  }
  int stage = 0;
  for (int c = mine; c < chunks; c += step) {
    const int ahead = c + (L::kStages - 1) * step;
    const int next = stage == 0 ? L::kStages - 1 : stage - 1;
    if (ahead < chunks) fetch(ahead, next);
    cp_async_commit();
    cp_async_wait<L::kStages - 1>();
    __syncwarp();
    const uint32_t ks = stage0 + stage * 2 * L::kTile, vs = ks + L::kTile;
    float s[KC / 8][4];
#pragma unroll
    for (int j = 0; j < KC / 8; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        uint32_t f[4];
        ldmatrix4(ks + (8 * j + (lane & 7)) * L::kPitch + (32 * d + (lane >> 3) * 8) * 2, f);
        mma16816<E>(s[j], qa[2 * d], f[0], f[1]);
        mma16816<E>(s[j], qa[2 * d + 1], f[2], f[3]);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < KC / 8; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = c * KC + 8 * j + (lane & 3) * 2 + (u & 1);
        s[j][u] = i < n ? s[j][u] * c2 : -INFINITY;
        top[u >> 1] = fmaxf(top[u >> 1], s[j][u]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      top[r] = fmaxf(top[r], m[r]);
      const float base = top[r] == -INFINITY ? 0.f : top[r];
      const float f = exp2f(m[r] - base);  // 0 at the first chunk
      l[r] *= f;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) o[i][2 * r] *= f, o[i][2 * r + 1] *= f;
      m[r] = top[r];
#pragma unroll
      for (int j = 0; j < KC / 8; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float& x = s[j][2 * r + u];
          x = ex2_approx(x - base);
          l[r] += x;
        }
    }
#pragma unroll
    for (int k = 0; k < KC / 16; ++k) {
      // P as the A operand in two parts of the input type, the rounded value and the rounding of what is left: 16 bits of
      // bf16, 22 of fp16. One part alone put 2.2e-3 of its norm into a bf16 result (its own rounding 1.65e-3), and with the
      // cache as the bound the second costs little: 174 against 171 us for 64 sequences, 74 against 70 for the one of 65,536.
      uint32_t a[4], rest[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x = s[2 * k + (u >> 1)][2 * (u & 1)], y = s[2 * k + (u >> 1)][2 * (u & 1) + 1];
        a[u] = pack2<E>(x, y);
        const float2 r = unpack2<E>(a[u]);
        rest[u] = pack2<E>(x - r.x, y - r.y);
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        uint32_t f[4];
        ldmatrix4_trans(vs + (16 * k + (lane & 15)) * L::kPitch + (16 * d + (lane >> 4) * 8) * 2, f);
        mma16816<E>(o[2 * d], a, f[0], f[1]);
        mma16816<E>(o[2 * d + 1], a, f[2], f[3]);
        mma16816<E>(o[2 * d], rest, f[0], f[1]);
        mma16816<E>(o[2 * d + 1], rest, f[2], f[3]);
      }
    }
    __syncwarp();  // the stage is free for the copies of the next step
    stage = stage == L::kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }

  // the warps' rows, [warp][row][DP + (m, l)], then the CTA's in the same form behind them
  __syncthreads();
  float* mine_rows = reinterpret_cast<float*>(smem) + warp * 16 * L::kRowFloats;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float* row = mine_rows + (lane / 4 + 8 * r) * L::kRowFloats;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
      *reinterpret_cast<float2*>(row + 8 * i + (lane & 3) * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    if ((lane & 3) == 0) row[DP] = m[r], row[DP + 1] = l[r];
  }
  __syncthreads();
  float* cta = reinterpret_cast<float*>(smem) + L::kWarps * 16 * L::kRowFloats;
  const float* rows = reinterpret_cast<const float*>(smem);
  for (int e = tid; e < heads * DP; e += L::kThreads) {
    const int r = e / DP, d = e % DP;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < L::kWarps; ++w) top = fmaxf(top, rows[(w * 16 + r) * L::kRowFloats + DP]);
    const float base = top == -INFINITY ? 0.f : top;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < L::kWarps; ++w) {
      const float* row = rows + (w * 16 + r) * L::kRowFloats;
      const float f = exp2f(row[DP] - base);
      acc = fmaf(row[d], f, acc), sum = fmaf(row[DP + 1], f, sum);
    }
    cta[r * L::kRowFloats + d] = acc;
    if (d == 0) cta[r * L::kRowFloats + DP] = top, cta[r * L::kRowFloats + DP + 1] = sum;
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  // the cluster's CTAs share out the (row, column) pairs of the result
  E* out = reinterpret_cast<E*>(p.out) + ((int64_t)b * p.H + head0) * p.D;
  for (int e = rank * L::kThreads + tid; e < heads * (DP / 2); e += parts * L::kThreads) {
    const int r = e / (DP / 2), d = (e % (DP / 2)) * 2;
    const float* row = cta + r * L::kRowFloats;
    float top = -INFINITY, mm[kMost], ll[kMost], x[kMost], y[kMost];
    if (parts == 1) {
      mm[0] = row[DP], ll[0] = row[DP + 1], x[0] = row[d], y[0] = row[d + 1];
      top = mm[0];
    } else {
#pragma unroll
      for (int k = 0; k < kMost; ++k) {
        if (k >= parts) break;
        const uint32_t at = cluster_addr(row, (uint32_t)k);
        mm[k] = ld_cluster_f32(at + DP * 4), ll[k] = ld_cluster_f32(at + DP * 4 + 4);
        x[k] = ld_cluster_f32(at + d * 4), y[k] = ld_cluster_f32(at + d * 4 + 4);
        top = fmaxf(top, mm[k]);
      }
    }
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, ax = 0.f, ay = 0.f;
#pragma unroll
    for (int k = 0; k < kMost; ++k) {
      if (k >= parts) break;
      const float f = exp2f(mm[k] - base);
      sum = fmaf(ll[k], f, sum), ax = fmaf(x[k], f, ax), ay = fmaf(y[k], f, ay);
    }
    const bool have = n > 0;
    const float inv = have ? 1.0f / sum : 0.f;
    if (d < p.D)
      *reinterpret_cast<uint32_t*>(out + (int64_t)r * p.D + d) = have ? pack2<E>(ax * inv, ay * inv) : 0u;
    if (d == 0 && p.lse)
      p.lse[(int64_t)b * p.H + head0 + r] = have ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  }
  if (parts > 1) cluster_sync();  // no CTA leaves while another reads its rows
}

int check_window(const NoiseWindow* a, bool token);

// CTAs per (sequence, key head), a power of two: as many as the two an SM holds take in at once (twice that from one
// CTA to two), as long as every warp gets a chunk; 16 only where they find an SM each and every warp still has eight
// chunks. Twice the CTAs against these: 8 sequences of 8,192 tokens, 8 key heads of 128, 72 against 65 us; 16 of 1,024 visible
// ones, 8 of 64, 20 against 16; but 32 of 4,096, 8 of 128, 108 against 116 with one. 8 against 16: one of 65,536, 8 of 128,
// 96 against 76; one of 16,384, 2 of 64, 20 against 16; but one of 4,096, 8 of 128, 14 against 16, two of 8,192 27 against 37.
static int token_ctas(const NoiseWindow* a, int sms, int widest) {
  const int window = a->window < a->Tk ? a->window : a->Tk, sinks = a->sinks < a->Tk ? a->sinks : a->Tk;
  const int64_t pairs = (int64_t)a->B * a->Hk * ((a->H / a->Hk + 15) / 16);
  const int64_t keys = (int64_t)window + 1 + sinks < a->Tk ? (int64_t)window + 1 + sinks : a->Tk;
  const int64_t chunks = a->D <= 64 ? WinTok<64>::kWarps * WinTok<64>::KC : WinTok<128>::kWarps * WinTok<128>::KC;
  int parts = 1;
  while (parts < 8 && pairs * parts <= (parts == 1 ? 2 : 1) * (int64_t)sms && keys > parts * chunks) parts *= 2;
  return parts == 8 && widest >= 16 && pairs * 16 <= sms && keys >= 16 * chunks * 8 ? 16 : parts;
}

template <typename E, int DP, int kMost>
static int launch_window_token(const TokenParams& p, int B, int Hk, int parts, cudaStream_t s) {
  using L = WinTok<DP>;
  static KernelOptIn opt_in;
  if (!opt_in(window_token_kernel<E, DP, kMost>, L::kSmem, kMost > 8)) return kStatusLaunchFailed;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)parts, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)parts, (unsigned)(Hk * p.tiles), (unsigned)B), cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmem, cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = parts > 1;
  if constexpr (kMost > 8) {  // more CTAs than every device places: asked for once a device
    static std::atomic<uint64_t> placed{0}, not_placed{0};
    int dev = 0, clusters = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return kStatusLaunchFailed;
    const uint64_t bit = 1ull << (dev & 63);
    if (!((placed.load() | not_placed.load()) & bit)) {
      if (cudaOccupancyMaxActiveClusters(&clusters, window_token_kernel<E, DP, kMost>, &cfg) != cudaSuccess)
        cudaGetLastError(), clusters = 0;
      (clusters > 0 ? placed : not_placed).fetch_or(bit);
    }
    if (not_placed.load() & bit) return kStatusUnsupported;
  }
  LaunchScope scope(kKindAttention, s);
  if (cudaLaunchKernelEx(&cfg, window_token_kernel<E, DP, kMost>, p) != cudaSuccess) {
    cudaGetLastError();
    return kStatusLaunchFailed;
  }
  return kStatusOk;
}

template <typename E, int DP>
static int launch_window_token(const NoiseWindow* a, cudaStream_t s) {
  using L = WinTok<DP>;
  TokenParams p{};
  p.q = a->q, p.k = a->k, p.v = a->v;
  p.q_b = a->q_stride[0], p.q_h = a->q_stride[2];
  p.k_b = a->k_stride[0], p.k_t = a->k_stride[1], p.k_h = a->k_stride[2];
  p.v_b = a->v_stride[0], p.v_t = a->v_stride[1], p.v_h = a->v_stride[2];
  p.lengths = a->lengths, p.out = a->out, p.lse = a->lse;
  p.H = a->H, p.group = a->H / a->Hk, p.tiles = (p.group + 15) / 16, p.Tk = a->Tk, p.D = a->D;
  p.window = a->window < a->Tk ? a->window : a->Tk, p.sinks = a->sinks < a->Tk ? a->sinks : a->Tk;
  p.scale = a->scale;
  if ((int64_t)a->Hk * p.tiles > 65535) return kStatusUnsupported;
  const int sms = device_sm_count(), parts = token_ctas(a, sms, 16);
  if (parts > 8) {
    const int rc = launch_window_token<E, DP, 16>(p, a->B, a->Hk, parts, s);
    if (rc != kStatusUnsupported) return rc;
  }
  return launch_window_token<E, DP, 8>(p, a->B, a->Hk, token_ctas(a, sms, 8), s);
}

}  // namespace noise

using namespace noise;

extern "C" int noise_window_token_ctas(const NoiseWindow* a, int sms, int widest) {
  const int rc = check_window(a, true);
  return rc != kStatusOk || a->B == 0 || sms < 1 ? -1 : token_ctas(a, sms, widest);
}

extern "C" int noise_window_token(const NoiseWindow* a, void* stream) {
  const int rc = check_window(a, true);
  if (rc != kStatusOk || a->B == 0) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == NOISE_BF16)
    return a->D <= 64 ? launch_window_token<__nv_bfloat16, 64>(a, s) : launch_window_token<__nv_bfloat16, 128>(a, s);
  return a->D <= 64 ? launch_window_token<__half, 64>(a, s) : launch_window_token<__half, 128>(a, s);
}
