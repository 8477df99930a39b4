// Causal attention with a sliding window and a few first tokens (sinks) that stay visible to every later
// query, on the 5th-generation tensor cores, for any length, grouped heads and padded batches:
//
//   S = scale Q K^T where visible, -inf elsewhere,   O = softmax(S) V,   lse = log sum exp S
//
// One pass over the keys: each query row keeps a reference m and the sum l of exp(S - m). m is the maximum of
// the first tile the row sees, and is raised only when a later tile's P sums to more than 2^10 under it; then
// the tile is taken again under its new maximum and O (in tensor memory) and l are scaled by exp(m_old - m_new).
// The sum that l needs anyway thus guards the range, and the usual tile spends no instruction on a maximum. P, l
// and O only meet as P / l and O / l, so a reference below the maximum costs no accuracy.
//
// One CTA = two consecutive tiles of 128 queries of one head; they share every key and value tile the CTA
// streams, while one tile's products overlap the other's exponentials. Key tiles: the sinks' first, then
// those the window reaches; 32 x 32 blocks of scores are skipped, taken without masks, or masked by a word of
// visible keys.
//   warp 0       TMA producer: Q once, then K and V tiles on rings of their own
//   warp 1       tensor memory owner and MMA issuer: per key tile and query tile, O += P V of the tile before,
//                then S = Q K^T (S reuses the columns that P lay in)
//   warps 2 ..   one query row a thread: S from tensor memory, the softmax step, P back over S as 16-bit pairs
// The head width is padded to 64 or 128 by the tensor maps' zero fill. At 64 (key tiles of 64, 256 columns of
// tensor memory) two CTAs share an SM; at 128 (key tiles of 128) one CTA takes all 512 columns.
//
// Measured at B 8, T 2048, 8 heads of 64, window 1024, 4 sinks (bf16) and at T 16384, 16 heads on 4 key heads of
// 128, window 4096, 64 sinks (fp16), in calls one after the other: 59 and 537 us, 435 and 907 TFLOP/s of visible pairs (the
// long one slows the clock: 479 us in a few calls at 1,965 MHz). The bound is the chain S -> softmax -> P -> O of each tile
// and the products' rate: without any softmax work the same pipeline takes 53 and 377 us (the latter at 1,965 MHz), and
// the products alone 31 and 305 us at their measured rates (43 + N / 2 cycles for 16 values of the inner dimension with
// both operands in shared memory, 11 + N / 2 with A in tensor memory). What other choices took, block and long prompt,
// each against the kernel as it was then, in a few calls:
//   a maximum of every tile: 153 against 102 us (both with the products issued from a one-lane branch)
//   P in columns of its own beside S, one CTA an SM at 64: 84 and 551 against 76 and 504
//   CTAs in launch order, not the heavy ones first: 76 and 504 against 64 and 479
//   at 128, P handed over 64 keys at a time: 493 against 479; two warps a row: 494
//   a quarter of the exponentials as polynomials on the fp32 units: 65 and 481 against 65 and 480
// P is rounded to the input type, as the tensor core needs it; the row sum is of the unrounded values. The result is then
// off by 2.1e-3 of its norm in bf16 and 2.5e-4 in fp16, where its own rounding makes 1.6e-3 and 2.0e-4. A second product
// with what the rounding left takes the difference away (1.6e-3, 2.0e-4) and 76 and 698 us: eight softmax warps have to
// split and store twice as much. Not kept for a part below the result's own rounding.
//
// A key tile that crosses the end of a padded sequence is loaded apart: the producer warp clears the value
// rows behind the end before the products see them, since 0 times a NaN is not 0. Every wait is bounded.
#include <type_traits>

#include "profile.cuh"
#include "window.cuh"

namespace noise {

// head width DP (64 or 128), key tile KT, G query tiles per CTA
template <int DP>
struct WinFwd {
  static constexpr int G = 2, kQ = 128;
  static constexpr int KT = DP == 64 ? 64 : 128;
  static constexpr int kThreads = (2 + 4 * G) * 32;
  static constexpr int kQBytes = kQ * DP * 2, kTileBytes = KT * DP * 2;
  static constexpr int KS = DP == 64 ? 3 : 2, VS = 2;
  static constexpr int kCore = G * kQBytes + (KS + VS) * kTileBytes;
  static constexpr int kSmem = 1024 + kCore + 256;
  static constexpr uint32_t kGroupCols = KT + DP;
  static constexpr uint32_t kTmemCols = DP == 64 ? 256 : 512;
  static constexpr int kCtas = DP == 64 ? 2 : 1;
};

// Sum of a tile's P above which the tile is taken again under a higher maximum. A tile under its own maximum sums
// to at most 128, so anything above says that the maximum has grown; up to 2^10 P stays exact enough in bf16 and
// fp16 (below 65,504) and the fp32 sums far from overflow.
constexpr float kWinTileSum = 1024.f;

// The key tiles of a CTA: sink tiles [0, sink), then tiles lo .. hi.
struct KeyWalk {
  int sink, lo, n;
  __device__ __forceinline__ int tile(int t) const { return t < sink ? t : lo + t - sink; }
};

template <typename E, int DP>
__global__ void __launch_bounds__(WinFwd<DP>::kThreads, WinFwd<DP>::kCtas)
    window_forward_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WindowParams p,
                          const __grid_constant__ TileOrder order) {
  using L = WinFwd<DP>;
  constexpr int G = L::G, KT = L::KT, KS = L::KS, VS = L::VS, kQ = L::kQ;
  constexpr uint32_t kFmt = std::is_same<E, __half>::value ? 0 : 1;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int unit, pair;
  order.at(blockIdx.x, unit, pair);
  unit = order.tiles - 1 - unit;  // longest key ranges first
  const int b = pair / p.H, head = pair - b * p.H, kv = head / p.group;
  const int i0 = unit * kQ * G;                 // first query row of the CTA
  const int length = window_length(p, b);
  const int rows = min(p.Tq, length - p.offset);  // query rows with a token
  E* out = reinterpret_cast<E*>(p.out);
  const int64_t row_elems = (int64_t)p.H * p.D;
  auto out_row = [&](int i) { return out + ((int64_t)b * p.Tq + i) * row_elems + (int64_t)head * p.D; };
  auto lse_at = [&](int i) { return p.lse + ((int64_t)b * p.H + head) * p.Tq + i; };
  if (i0 >= rows) {  // padding only
    const int n = min(kQ * G, p.Tq - i0);
    for (int e = tid; e < n * (p.D / 8); e += L::kThreads) {
      const int r = e / (p.D / 8), c = e - r * (p.D / 8);
      *reinterpret_cast<uint4*>(out_row(i0 + r) + 8 * c) = make_uint4(0u, 0u, 0u, 0u);
    }
    for (int r = tid; r < n; r += L::kThreads) *lse_at(i0 + r) = -INFINITY;
    return;
  }
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* sK = sQ + G * L::kQBytes;
  uint8_t* sV = sK + KS * L::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::kCore);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;    // [KS]
  uint64_t* k_empty = k_full + KS;  // [KS]
  uint64_t* v_full = k_empty + KS;  // [VS]
  uint64_t* v_empty = v_full + VS;  // [VS]
  uint64_t* s_full = v_empty + VS;  // [G]
  uint64_t* p_full = s_full + G;    // [G]
  uint64_t* o_full = p_full + G;    // [G]
  uint64_t* tail = o_full + G;      // the value tile that crosses the sequence's end
  uint64_t* drain = tail + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int active = rows - i0 > kQ ? 2 : 1;  // query tiles with a token
  auto q_first = [&](int g) { return p.offset + i0 + kQ * g; };
  auto q_last = [&](int g) { return min(p.offset + i0 + kQ * g + kQ, length) - 1; };
  auto tile_lo = [&](int g) { return max(0, q_first(g) - p.window) / KT; };
  auto tile_hi = [&](int g) { return q_last(g) / KT; };
  const int sink_tiles = (p.sinks + KT - 1) / KT;
  KeyWalk walk;
  walk.lo = tile_lo(0);
  walk.sink = min(sink_tiles, walk.lo);
  walk.n = walk.sink + tile_hi(active - 1) - walk.lo + 1;
  const int lo0 = walk.lo, hi0 = tile_hi(0), lo1 = tile_lo(1), hi1 = tile_hi(1);
  auto needs = [&](int g, int kt) {
    return kt <= (g ? hi1 : hi0) && (kt >= (g ? lo1 : lo0) || kt < sink_tiles);
  };
  int* status = p.status;

  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < KS; ++s) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 1);
    for (int s = 0; s < VS; ++s) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 1);
    for (int g = 0; g < G; ++g) mbar_init(&s_full[g], 1), mbar_init(&p_full[g], 4), mbar_init(&o_full[g], 1);
    mbar_init(tail, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer (the whole warp: it clears rows of the tile that crosses the end) --------
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, active * L::kQBytes);
      for (int g = 0; g < active; ++g)
        for (int c = 0; c < DP / 64; ++c)
          tma_load_4d(sQ + g * L::kQBytes + c * (kQ * 128), &tm_q, q_full, 64 * c, head, i0 + kQ * g, b);
    }
    int nk = 0, nv = 0;
    bool ok = true;
    auto all_lanes = [](bool v) { return __all_sync(0xffffffffu, v) != 0; };
    auto load = [&](bool key, int t) {  // the lanes leave together, whatever a wait returned to each
      const int stages = key ? KS : VS, st = t % stages, kt = walk.tile(t);
      uint64_t* full = key ? &k_full[st] : &v_full[st];
      if (!all_lanes(mbar_wait(key ? &k_empty[st] : &v_empty[st], ((t / stages) & 1) ^ 1, abort_flag, status)))
        return false;
      const int behind = (kt + 1) * KT - length;  // rows of the tile behind the sequence's end
      const bool clear = !key && behind > 0 && length < p.Tk;
      uint8_t* dst = (key ? sK : sV) + st * L::kTileBytes;
      if (lane == 0) {
        uint64_t* bar = clear ? tail : full;
        mbar_arrive_expect_tx(bar, L::kTileBytes);
        for (int c = 0; c < DP / 64; ++c)
          tma_load_4d(dst + c * (KT * 128), key ? &tm_k : &tm_v, bar, 64 * c, kv, kt * KT, b);
      }
      if (clear) {
        if (!all_lanes(mbar_wait(tail, 0, abort_flag, status))) return false;
        for (int c = 0; c < DP / 64; ++c) {  // whole 128-byte rows: the swizzle stays inside a row
          uint4* at = reinterpret_cast<uint4*>(dst + c * (KT * 128) + (KT - behind) * 128);
          for (int e = lane; e < behind * 8; e += 32) at[e] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
      }
      return true;
    };
    while (ok && nv < walk.n) {
      if (nk < walk.n && nk < nv + KS - 1) ok = load(true, nk++);
      else ok = load(false, nv++);
    }
    if (lane == 0) {  // copies in flight land before the CTA can exit
      mbar_wait(q_full, 0, abort_flag, status);
      for (int j = max(0, nk - KS); j < nk; ++j) mbar_wait(&k_full[j % KS], (j / KS) & 1, abort_flag, status);
      for (int j = max(0, nv - VS); j < nv; ++j) mbar_wait(&v_full[j % VS], (j / VS) & 1, abort_flag, status);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // The whole warp walks the loop, so that descriptors and addresses are warp-uniform values; one elected lane
    // issues. (From inside a one-lane branch every product waits for its operands to reach uniform registers,
    // about 100 cycles.)
    const uint32_t idesc_s = make_idesc(kFmt, kQ, KT);
    const uint32_t idesc_o = make_idesc(kFmt, kQ, DP, 0, 1);  // B = V is MN-major
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const bool issuer = elect_one();
    int np[G] = {0, 0};                                       // PV products issued
    bool need[G] = {false, false};                            // which query tiles the tile before is for
    bool ok = mbar_wait_warp(q_full, 0, abort_flag, status);
    for (int t = 0; ok && t <= walk.n; ++t) {
      bool now[G] = {false, false};
      const int ks = t % KS, vs = (t + VS - 1) % VS;  // stages of this tile's keys and the last tile's values
      if (t < walk.n) {
        const int kt = walk.tile(t);
        now[0] = needs(0, kt), now[1] = active > 1 && needs(1, kt);
        if (!(ok = mbar_wait_warp(&k_full[ks], (t / KS) & 1, abort_flag, status))) break;
      }
      if (t > 0 && !(ok = mbar_wait_warp(&v_full[vs], ((t - 1) / VS) & 1, abort_flag, status))) break;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t tS = tm + L::kGroupCols * g;
        if (ok && need[g]) {
          ok = mbar_wait_warp(&p_full[g], np[g] & 1, abort_flag, status);
          if (ok) {
            tc_fence_after();
            if (issuer) {
              const uint64_t dv = smem_desc_sw128_mn(sV + vs * L::kTileBytes, KT * 128);
#pragma unroll
              for (int k = 0; k < KT / 16; ++k)
                tc_mma_f16_ts(tS + KT, tS + 8 * k, dv + (uint64_t)(2048 >> 4) * k, idesc_o, (np[g] > 0 || k > 0) ? 1u : 0u);
              if (walk.tile(t - 1) == (g ? hi1 : hi0)) tc_commit(&o_full[g]);
            }
            ++np[g];
          }
        }
        if (ok && now[g]) {
          tc_fence_after();
          if (issuer) {
            const uint64_t dq = smem_desc_sw128(sQ + g * L::kQBytes), dk = smem_desc_sw128(sK + ks * L::kTileBytes);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
              tc_mma_f16(tS, dq + (k / 4) * (kQ * 128 >> 4) + 2 * (k % 4),
                         dk + (k / 4) * (KT * 128 >> 4) + 2 * (k % 4), idesc_s, k > 0 ? 1u : 0u);
            tc_commit(&s_full[g]);
          }
        }
      }
      if (!ok) break;
      if (issuer) {
        if (t > 0) tc_commit(&v_empty[vs]);
        if (t < walk.n) tc_commit(&k_empty[ks]);
      }
      need[0] = now[0], need[1] = now[1];
    }
    if (issuer) {
      tc_commit(drain);
      mbar_wait(drain, 0, abort_flag, status);
    }
    __syncwarp();
  } else {
    // ---------------- softmax and output ----------------
    const int g = (warp - 2) >> 2, quarter = warp & 3;
    const int i = i0 + kQ * g + quarter * 32 + lane;  // query row of this thread
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + L::kGroupCols * g + lanes, tO = tS + KT;
    if (g < active) {
      const float c = p.scale * 1.4426950408889634f;
      const float2 c2 = make_float2(c, c);
      const int q = p.offset + i;
      const int qlo = q_first(g) + quarter * 32, qhi = qlo + 31;  // this warp's positions
      float m = -INFINITY;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      bool ok = true;
      int n = 0;
      for (int t = 0; t < walk.n; ++t) {
        const int kt = walk.tile(t);
        if (!needs(g, kt)) continue;
        if (!(ok = mbar_wait_warp(&s_full[g], n & 1, abort_flag, status))) break;
        tc_fence_after();
        const int k0 = kt * KT;
        // P of the tile, with m as it stands; `raise` (for the whole warp) first lifts m to the rows' maxima
        bool raise = !__all_sync(0xffffffffu, m > -INFINITY);
        uint32_t w[KT / 2];
        float2 t2[2];
        while (true) {
          if (raise) {
            float top = -INFINITY;
#pragma unroll 1
            for (int h = 0; h < KT / 32; ++h) {
              const int kc = k0 + 32 * h;
              if (window_none(qlo, qhi, kc, kc + 31, p.window, p.sinks)) continue;
              float sv[32];
              tmem_read32(tS + 32 * h, sv);
              const uint32_t seen = window_keys(q, kc, p.window, p.sinks);
#pragma unroll
              for (int u = 0; u < 32; ++u)
                if (seen >> u & 1) top = fmaxf(top, sv[u]);
            }
            const float next = fmaxf(m, top * c);
            const float f = next > m ? exp2f(m - next) : 1.f;  // 0 for the row's first visible key
            m = next;
            sum[0].x *= f, sum[0].y *= f, sum[1].x *= f, sum[1].y *= f;
            if (n > 0) {  // the products before this S have completed: O is this warp's to change
#pragma unroll 1
              for (int h = 0; h < DP / 16; ++h) {
                uint32_t o[16];
                tmem_ld16(tO + 16 * h, o);
#pragma unroll
                for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                tmem_st16(tO + 16 * h, o);
              }
            }
          }
          const float off = m == -INFINITY ? 0.f : -m;
          const float2 off2 = make_float2(off, off);
          t2[0] = t2[1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int h = 0; h < KT / 32; ++h) {
            const int kc = k0 + 32 * h;
            if (window_none(qlo, qhi, kc, kc + 31, p.window, p.sinks)) {
#pragma unroll
              for (int u = 0; u < 16; ++u) w[16 * h + u] = 0u;
              continue;
            }
            float sv[32];
            tmem_read32(tS + 32 * h, sv);
            if (!window_all(qlo, qhi, kc, kc + 31, p.window, p.sinks)) {
              const uint32_t seen = window_keys(q, kc, p.window, p.sinks);
#pragma unroll
              for (int u = 0; u < 32; ++u)
                if (!(seen >> u & 1)) sv[u] = -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const float2 x = __ffma2_rn(make_float2(sv[2 * u], sv[2 * u + 1]), c2, off2);
              const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              t2[u & 1] = __fadd2_rn(t2[u & 1], e);
              w[16 * h + u] = pack2<E>(e.x, e.y);
            }
          }
          if (raise) break;
          const float t = (t2[0].x + t2[0].y) + (t2[1].x + t2[1].y);
          if (__all_sync(0xffffffffu, t <= kWinTileSum)) break;
          raise = true;
        }
        sum[0] = __fadd2_rn(sum[0], t2[0]), sum[1] = __fadd2_rn(sum[1], t2[1]);
#pragma unroll
        for (int h = 0; h < KT / 32; ++h) tmem_st16(tS + 16 * h, *reinterpret_cast<uint32_t(*)[16]>(w + 16 * h));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
        ++n;
      }
      if (ok && mbar_wait_warp(&o_full[g], 0, abort_flag, status)) {
        tc_fence_after();
        const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        const bool have = i < rows;
        const float inv = have ? 1.0f / l : 0.f;
#pragma unroll
        for (int h = 0; h < DP / 32; ++h) {
          float o[32];
          tmem_read32(tO + 32 * h, o);
          if (i >= p.Tq) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (32 * h + 8 * u >= p.D) break;
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              w[x] = have ? pack2<E>(o[8 * u + 2 * x] * inv, o[8 * u + 2 * x + 1] * inv) : 0u;
            st_global_v4(out_row(i) + 32 * h + 8 * u, w[0], w[1], w[2], w[3]);
          }
        }
        if (i < p.Tq) *lse_at(i) = have ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
      }
    } else if (i < p.Tq) {  // a tile of padding beside one with tokens
      for (int u = 0; u < p.D / 8; ++u) st_global_v4(out_row(i) + 8 * u, 0u, 0u, 0u, 0u);
      *lse_at(i) = -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <typename E, int DP>
static int launch_window_forward(const NoiseWindow* a, const WindowParams& p, cudaStream_t s) {
  using L = WinFwd<DP>;
  static KernelOptIn opt_in;
  CUtensorMap tq, tk, tv;
  if (make_tmap_bthd(&tq, a->q, a->dtype, a->B, a->Tq, a->H, a->D, a->q_stride, L::kQ) ||
      make_tmap_bthd(&tk, a->k, a->dtype, a->B, a->Tk, a->Hk, a->D, a->k_stride, L::KT) ||
      make_tmap_bthd(&tv, a->v, a->dtype, a->B, a->Tk, a->Hk, a->D, a->v_stride, L::KT))
    return kStatusBadArgument;
  if (!opt_in(window_forward_kernel<E, DP>, L::kSmem)) return kStatusLaunchFailed;
  const int64_t units = (a->Tq + L::kQ * L::G - 1) / (L::kQ * L::G), pairs = (int64_t)a->B * a->H;
  if (units * pairs > INT32_MAX) return kStatusUnsupported;
  const TileOrder order = tile_order((int)units, (int)pairs, (int64_t)a->Tk * a->D * 4 / p.group);
  LaunchScope scope(kKindAttention, s);
  window_forward_kernel<E, DP><<<(unsigned)(units * pairs), L::kThreads, L::kSmem, s>>>(tq, tk, tv, p, order);
  return cudaGetLastError() == cudaSuccess ? kStatusOk : kStatusLaunchFailed;
}

bool window_operand_ok(const void* ptr, const int64_t* stride, int B, int T, int heads) {
  if (!ptr || !is_aligned(ptr, 16)) return false;
  const int64_t n[3] = {B, T, heads};
  for (int i = 0; i < 3; ++i) {
    // a dimension of one element is never stepped along; others need a positive step of whole 16 bytes
    if (n[i] > 1 && (stride[i] <= 0 || stride[i] % 8 || stride[i] >= (1ll << 39))) return false;
  }
  return true;
}

int check_window(const NoiseWindow* a, bool token) {
  if (!a || a->B < 0 || a->Tk < 1 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->window < 0 || a->sinks < 0 ||
      !(a->scale >= 0x1p-100f && a->scale <= 0x1p100f))
    return kStatusBadArgument;
  if (a->dtype != NOISE_BF16 && a->dtype != NOISE_FP16) return kStatusUnsupported;
  if (a->D < 8 || a->D > 128 || a->D % 8) return kStatusUnsupported;
  if (a->B > 65535 || a->H > 65535 || a->Tk > (1 << 30)) return kStatusUnsupported;
  if (a->B == 0) return kStatusOk;
  if (!token) {
    if (a->Tq < 1 || a->offset < 0 || a->offset > a->Tk - a->Tq) return kStatusBadArgument;
    if (!window_operand_ok(a->q, a->q_stride, a->B, a->Tq, a->H) || !a->lse) return kStatusBadArgument;
  } else {
    if (!window_operand_ok(a->q, a->q_stride, a->B, 1, a->H) || !a->lengths) return kStatusBadArgument;
  }
  if (!window_operand_ok(a->k, a->k_stride, a->B, a->Tk, a->Hk) ||
      !window_operand_ok(a->v, a->v_stride, a->B, a->Tk, a->Hk) || !a->out || !is_aligned(a->out, 16))
    return kStatusBadArgument;
  return kStatusOk;
}

WindowParams window_params(const NoiseWindow* a, int* status) {
  WindowParams p{};
  p.B = a->B, p.Tq = a->Tq, p.Tk = a->Tk, p.H = a->H, p.group = a->H / a->Hk, p.D = a->D, p.offset = a->offset;
  // a window of Tk keys sees everything; the clamp keeps differences of positions inside 32 bits
  p.window = a->window < a->Tk ? a->window : a->Tk, p.sinks = a->sinks < a->Tk ? a->sinks : a->Tk;
  p.scale = a->scale, p.lengths = a->lengths, p.out = a->out, p.lse = a->lse, p.status = status;
  return p;
}

}  // namespace noise

using namespace noise;

extern "C" int noise_window_attention(const NoiseWindow* a, int* status, void* stream) {
  const int rc = check_window(a, false);
  if (rc != kStatusOk) return rc;
  if (!status) return kStatusBadArgument;
  if (a->B == 0) return kStatusOk;
  const WindowParams p = window_params(a, status);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == NOISE_BF16)
    return a->D <= 64 ? launch_window_forward<__nv_bfloat16, 64>(a, p, s) : launch_window_forward<__nv_bfloat16, 128>(a, p, s);
  return a->D <= 64 ? launch_window_forward<__half, 64>(a, p, s) : launch_window_forward<__half, 128>(a, p, s);
}
