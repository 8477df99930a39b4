// Gradient of the sliding-window attention with sinks (window_attention.cu). With P = exp(scale Q K^T - lse) on
// the visible pairs, which the saved lse gives back without a second pass over the row:
//
//   Delta_i = sum_d dO_id O_id,   dP = dO V^T,   dS = P * (dP - Delta)
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K
//
// Two launches (more where a key tile's queries are split):
//   window_stats:    Delta, and -lse in base 2, of every query row, in chunks of 64 rows the others load whole.
//   window_backward: the keys' side, one CTA = 128 keys, streaming the 64-query tiles of every head of the group that
//                    see them; then the queries' side, one CTA = 128 queries of one head, streaming the 64-key tiles.
// S and dP are formed on both sides, and dS goes into dQ and dK in two parts (below): 9 products a block of pairs where
// the formulas have 5, and one of 16 columns for the addends. Every gradient is so summed in one CTA's tensor memory in a
// fixed order. Adding dQ across key tiles with atomics would save S and dP a second time and make the result depend on
// timing.
//
// The sides have one body. X0, X1 are the CTA's own 128-row tiles, Y0, Y1 the streamed 64-row tiles:
//   S  = X0 Y0^T, dP = X1 Y1^T  (X in shared memory on the keys' side, in tensor memory, where its product is faster,
//                                on the queries' side, which has columns left; accumulators in tensor memory)
//   P and dS, as 16-bit pairs over the columns that S and dP lay in, are the A operands of
//   keys' side (X = K, V; Y = Q, dO; rows are keys):     dV += P Y1, dK += dS Y0
//   queries' side (X = Q, dO; Y = K, V; rows are queries): dQ += dS Y0
// with Y0, Y1 read a second time, now as MN-major B operands, from the same shared memory. On the keys' side lse and
// Delta belong to columns: one more product, of rows of ones with their three bf16 parts (24 bits), puts -lse / scale
// under S and -Delta under dP. Read from shared memory by every thread instead they took turns with the tensor core's
// own reads: 240 us against 217.
//
// Measured (all launches) at B 8, T 2048, 8 heads of 64, window 1024, 4 sinks: 220 us, 294 TFLOP/s of the five products
// over the visible pairs; at 4 padded sequences of up to 1,999 tokens, 12 heads on 4 of 128, window 511, 16 sinks:
// 109 us. What bounds it is each item's chain (S and dP, the warps' arithmetic, the gradients' products) at 64, the
// products' rate and a CTA's first and last item at 128. So two items are in flight per SM (two CTAs with one buffer of
// S and dP each at 64, one CTA with two buffers at 128) and eight warps share an item, each with 32 rows and half of
// the columns. One persistent CTA an SM with P and dS beside S and dP: 197 and 125 against 211 and 100 us.
// P is rounded to bf16, as the tensor core needs: dV is off by 2.3e-3 of its norm (1.7e-3 with the rest of P in a second
// product, 235 against 220 us). dS goes in as two bf16 numbers, its upper half (cut, which costs one
// permute a pair; rounded, 235 against 227 us) and the rest rounded, 16 bits in all, in the columns that dP lay in:
// rounded to one, dQ and dK were off by 2.4e-3 of their norm where the rounding of the result alone makes 1.7e-3, and
// the kernel took 20 us less. Sums are fp32.
//
// Sinks are seen by every later query, so their key tiles have far more work than the others: it is dealt in
// chunks to several CTAs that write fp32 partial sums, added in order by a last launch. Grouped heads with few
// key tiles are split the same way. Rows of a streamed tile behind a padded sequence's end are cleared in
// shared memory before the products, since 0 times a NaN is not 0. Every wait is bounded.
#include "profile.cuh"
#include "window.cuh"

namespace noise {

struct WindowGrad {
  WindowParams w;
  const float* stat;  // [B, H, tiles][2][64]: -lse log2(e), then -Delta; padding rows hold (-inf, 0)
  const uint4* adds;  // [B, H, tiles][2][64]: -lse / scale, then -Delta, in three bf16 parts; padding rows hold zeros
  int stat_tiles;
  void *dq, *dk, *dv;  // contiguous [B, T, heads, D]
  float* partial;      // [slot][2][128][D] sums of split key tiles
  int sink_tiles, sink_splits, splits, slots;  // key tiles that hold sinks come first; slots per (sequence, key head)
  TileOrder keys, queries;
  const __nv_bfloat16 *q, *dout;  // element strides {batch, token, head}, 0 where a dimension has one element
  int64_t q_step[3], dout_step[3];
};

// Boxes of 128 rows for the keys' side's own tiles, of 64 for the streamed ones.
struct WindowMaps {
  CUtensorMap k128, v128, q64, o64, k64, v64;
};

// The addends of S and dP: rows of eight bf16, 64 rows each.
constexpr int kAddBytes = 2 * 64 * 16;

template <int DP>
struct WinBwd {
  static constexpr int kX = 128, kY = 64, YS = 3;
  static constexpr int NB = DP == 64 ? 1 : 2, kCtas = DP == 64 ? 2 : 1;
  static constexpr int kSets = 2 * NB;  // sets of four warps: each buffer's columns are shared by two
  static constexpr int kThreads = (2 + 4 * kSets) * 32;
  static constexpr int kXBytes = kX * DP * 2, kYBytes = kY * DP * 2, kStage = 2 * kYBytes;
  static constexpr int kAdds = (YS + 1) * 2 * kAddBytes;  // the streamed tiles' addends, ones; each with zeros behind it
  static constexpr int kCore = kAdds + 2 * kXBytes + YS * kStage;
  static constexpr int kSmem = 1024 + kCore + 256;
  static constexpr uint32_t kAcc = NB * 128;  // columns: NB x (S 64, dP 64), then the gradients
  static constexpr uint32_t kTmemCols = 512 / kCtas;
  static constexpr uint32_t kXCol = kAcc + DP;  // queries' side: Q, then dO, as 16-bit pairs
  static_assert(kAcc + 2 * DP <= kTmemCols, "S, dP and both gradients lie in tensor memory");
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// v as the sum of three bf16 numbers (24 bits), in the first places of a row of eight.
__device__ __forceinline__ uint4 three_parts(float v) {
  const __nv_bfloat16 a = __float2bfloat16_rn(v);
  const float rest = v - __bfloat162float(a);
  const __nv_bfloat16 b = __float2bfloat16_rn(rest);
  return make_uint4(__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16,
                    __bfloat16_as_ushort(__float2bfloat16_rn(rest - __bfloat162float(b))), 0u, 0u);
}

// Delta and -lse of 64 query rows of one head: D / 8 lanes a row, 16 bytes a lane.
__global__ void __launch_bounds__(256) window_stats_kernel(const __nv_bfloat16* __restrict__ o,
                                                           const __nv_bfloat16* __restrict__ g, int64_t g_b, int64_t g_t,
                                                           int64_t g_h, const __grid_constant__ WindowParams p,
                                                           float* __restrict__ stat, uint4* __restrict__ adds) {
  const int tile = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int rows = min(p.Tq, window_length(p, b) - p.offset);
  const int lane = threadIdx.x & 15, first = threadIdx.x >> 4;  // 16 lanes a row
  const int64_t at = (((int64_t)b * p.H + head) * gridDim.x + tile) * 128;
  float* out = stat + at;
#pragma unroll
  for (int r = first; r < 64; r += 16) {
    const int i = tile * 64 + r;
    float t = 0.f;
    if (i < rows && lane * 8 < p.D) {
      Vec8<__nv_bfloat16> a, c;
      a.load(o + (((int64_t)b * p.Tq + i) * p.H + head) * p.D + lane * 8);
      c.load(g + b * g_b + i * g_t + head * g_h + lane * 8);
      float x[8], y[8];
      a.get(x), c.get(y);
#pragma unroll
      for (int u = 0; u < 8; ++u) t = fmaf(x[u], y[u], t);
    }
#pragma unroll
    for (int s = 8; s; s >>= 1) t += __shfl_xor_sync(0xffffffffu, t, s);
    if (lane == 0) {
      const float lse = i < rows ? p.lse[((int64_t)b * p.H + head) * p.Tq + i] : 0.f;
      out[r] = i < rows ? -1.4426950408889634f * lse : -INFINITY;
      out[64 + r] = -t;
      adds[at + r] = three_parts(-lse / p.scale);
      adds[at + 64 + r] = three_parts(-t);
    }
  }
}

// One CTA of either side; `index` is its place in that side's order.
template <int DP, bool kKeys>
__device__ __forceinline__ void window_side(const WindowMaps& m, const WindowGrad& p, int index) {
  using L = WinBwd<DP>;
  constexpr int NB = L::NB, YS = L::YS, kX = L::kX, kY = L::kY;
  const CUtensorMap &tm_y0 = kKeys ? m.q64 : m.k64, &tm_y1 = kKeys ? m.o64 : m.v64;
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const WindowParams& w = p.w;
  const int heads_k = w.H / w.group;
  int place, pair;  // place: the keys' side's (tile, split), or the query tile from the last
  (kKeys ? p.keys : p.queries).at(index, place, pair);
  const int b = pair / (kKeys ? heads_k : w.H), own_head = pair - b * (kKeys ? heads_k : w.H);
  const int length = window_length(w, b);
  const int rows = min(w.Tq, length - w.offset);  // query rows with a token (may be <= 0)

  // this CTA's X tile and its items, each one streamed Y tile
  int x0, kv, head0, items, begin = 0, slot = -1;
  int first_y, per_head;             // keys' side: query tiles first_y .. of each head of the group
  int sink_y = 0;                    // queries' side: sink tiles [0, sink_y), then first_y ..
  if (kKeys) {
    int tile, split, splits;
    const int sink_places = p.sink_tiles * p.sink_splits;
    if (place < sink_places) {
      tile = place / p.sink_splits, split = place - tile * p.sink_splits, splits = p.sink_splits;
      if (splits > 1) slot = place;
    } else {
      const int r = place - sink_places;
      tile = p.sink_tiles + r / p.splits, split = r % p.splits, splits = p.splits;
      if (splits > 1) slot = (p.sink_splits > 1 ? sink_places : 0) + r;
    }
    if (slot >= 0) slot += pair * p.slots;
    x0 = tile * kX, kv = own_head, head0 = kv * w.group;
    const int last_key = min(x0 + kX, length) - 1;
    const int lo = max(0, x0 - w.offset);
    const int hi = x0 < w.sinks ? rows - 1 : min(rows - 1, last_key + w.window - w.offset);
    first_y = lo / kY;
    per_head = last_key >= x0 && hi >= lo ? hi / kY - first_y + 1 : 0;
    const int all = per_head * w.group, share = (all + splits - 1) / splits;
    begin = min(all, split * share);
    items = min(all, begin + share) - begin;
  } else {
    x0 = (p.queries.tiles - 1 - place) * kX, head0 = own_head, kv = head0 / w.group;
    first_y = per_head = items = 0;
    if (x0 < rows) {
      const int q_first = w.offset + x0, q_last = min(w.offset + x0 + kX, length) - 1;
      first_y = max(0, q_first - w.window) / kY;
      sink_y = min((w.sinks + kY - 1) / kY, first_y);
      items = sink_y + q_last / kY - first_y + 1;
    }
  }
  // A walk over the items: the Y tile and, on the keys' side, the query head of the item it stands at.
  struct Walk {
    int y, head;
  };
  auto step_to = [&](Walk& it, int t, int n) {  // n items further, to item t
    if (kKeys) {
      for (it.y += n; it.y >= first_y + per_head; it.y -= per_head) ++it.head;
    } else {
      it.y = t < sink_y ? t : first_y + t - sink_y;
    }
  };
  Walk it{first_y, kKeys ? head0 : 0};

  __nv_bfloat16* g0 = reinterpret_cast<__nv_bfloat16*>(kKeys ? p.dk : p.dq);
  __nv_bfloat16* g1 = reinterpret_cast<__nv_bfloat16*>(p.dv);
  const int T = kKeys ? w.Tk : w.Tq, heads = kKeys ? heads_k : w.H, head = kKeys ? kv : head0;
  auto grad_row = [&](__nv_bfloat16* g, int i) { return g + (((int64_t)b * T + i) * heads + head) * w.D; };

  if (items <= 0) {  // no pair: zeros
    if (slot >= 0) {
      float4* out = reinterpret_cast<float4*>(p.partial + (int64_t)slot * 2 * kX * w.D);
      for (int e = tid; e < 2 * kX * w.D / 4; e += L::kThreads) out[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      const int n = min(kX, T - x0), c = w.D / 8;
      for (int e = tid; e < n * c; e += L::kThreads) {
        const int64_t at = (e % c) * 8;
        *reinterpret_cast<uint4*>(grad_row(g0, x0 + e / c) + at) = make_uint4(0u, 0u, 0u, 0u);
        if (kKeys) *reinterpret_cast<uint4*>(grad_row(g1, x0 + e / c) + at) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }

  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sAdd = base;                 // keys' side: [stage] addends, zeros; then ones, zeros
  uint8_t* sX = base + L::kAdds;        // X0, X1
  uint8_t* sY = sX + 2 * L::kXBytes;    // [stage] Y0, Y1
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::kCore);
  uint64_t* x_full = bars;
  uint64_t* y_full = x_full + 1;    // [YS]
  uint64_t* y_empty = y_full + YS;  // [YS]
  uint64_t* s_full = y_empty + YS;  // [NB]
  uint64_t* p_full = s_full + NB;   // [NB]
  uint64_t* tail = p_full + NB;     // a Y tile that crosses the end
  uint64_t* done = tail + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* status = w.status;
  if (tid == 0) {
    mbar_init(x_full, kKeys ? 1 : 8);
    for (int s = 0; s < YS; ++s) mbar_init(&y_full[s], 1), mbar_init(&y_empty[s], 1);
    for (int s = 0; s < NB; ++s) mbar_init(&s_full[s], 1), mbar_init(&p_full[s], 8);
    mbar_init(tail, 1);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    if (kKeys) prefetch_tensormap(&m.k128), prefetch_tensormap(&m.v128);
    prefetch_tensormap(&tm_y0);
    prefetch_tensormap(&tm_y1);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  if (kKeys) {  // rows (1, 1, 1, 0, ..) and the zeros behind every block
    for (int e = tid; e < kAddBytes / 16; e += L::kThreads) {
      reinterpret_cast<uint4*>(sAdd + YS * 2 * kAddBytes)[e] = make_uint4(0x3f803f80u, 0x3f80u, 0u, 0u);
#pragma unroll
      for (int j = 0; j <= YS; ++j) reinterpret_cast<uint4*>(sAdd + (2 * j + 1) * kAddBytes)[e] = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer (the whole warp) ----------------
    auto all_lanes = [](bool v) { return __all_sync(0xffffffffu, v) != 0; };
    if (kKeys && lane == 0) {
      mbar_arrive_expect_tx(x_full, 2 * L::kXBytes);
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_4d(sX + c * (kX * 128), &m.k128, x_full, 64 * c, head, x0, b);
        tma_load_4d(sX + L::kXBytes + c * (kX * 128), &m.v128, x_full, 64 * c, head, x0, b);
      }
    }
    const int end = kKeys ? rows : length, total = kKeys ? w.Tq : w.Tk;
    int t = 0, tails = 0;
    for (; t < items; ++t) {
      step_to(it, t, t == 0 ? begin : 1);
      const int st = t % YS, y0 = it.y * kY, hd = kKeys ? it.head : kv;
      if (!all_lanes(mbar_wait(&y_empty[st], ((t / YS) & 1) ^ 1, abort_flag, status))) break;
      const int behind = y0 + kY - end;
      const bool clear = behind > 0 && end < total;
      uint8_t* dst = sY + st * L::kStage;
      if (lane == 0) {
        uint64_t* bar = clear ? tail : &y_full[st];
        mbar_arrive_expect_tx(bar, L::kStage + (kKeys ? kAddBytes : 0));
        for (int c = 0; c < DP / 64; ++c) {
          tma_load_4d(dst + c * (kY * 128), &tm_y0, bar, 64 * c, hd, y0, b);
          tma_load_4d(dst + L::kYBytes + c * (kY * 128), &tm_y1, bar, 64 * c, hd, y0, b);
        }
        if (kKeys)
          bulk_load(sAdd + st * 2 * kAddBytes, p.adds + (((int64_t)b * w.H + hd) * p.stat_tiles + y0 / kY) * 128, kAddBytes, bar);
      }
      if (clear) {
        if (!all_lanes(mbar_wait(tail, tails & 1, abort_flag, status))) break;
        ++tails;
        for (int c = 0; c < 2 * (DP / 64); ++c) {  // whole 128-byte rows: the swizzle stays inside a row
          uint4* at = reinterpret_cast<uint4*>(dst + c * (kY * 128) + (kY - behind) * 128);
          for (int e = lane; e < behind * 8; e += 32) at[e] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&y_full[st]);
      }
    }
    if (lane == 0) {  // copies in flight land before the CTA can exit
      if (kKeys) mbar_wait(x_full, 0, abort_flag, status);
      for (int j = max(0, t - YS); j < t; ++j) mbar_wait(&y_full[j % YS], (j / YS) & 1, abort_flag, status);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (the whole warp, one elected lane issuing: see the forward) ----------------
    // Item t's S and dP, then the gradients of item t - 1: with two buffers, S(t) overwrites the
    // columns of P(t - 2), whose products were issued before it.
    const uint32_t idesc_s = make_idesc(1, kX, kY), idesc_g = make_idesc(1, kX, DP, 0, 1);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const bool issuer = elect_one();
    bool ok = mbar_wait_warp(x_full, 0, abort_flag, status);
    for (int t = 0; ok && t < items + NB - 1; ++t) {
      if (t < items) {
        const int st = t % YS, bf = t % NB;
        if (!(ok = mbar_wait_warp(&y_full[st], (t / YS) & 1, abort_flag, status))) break;
        tc_fence_after();
        const uint32_t tS = tm + 128 * bf;
        if (issuer) {
          const uint64_t x = smem_desc_sw128(sX), y = smem_desc_sw128(sY + st * L::kStage);
          if (kKeys)  // -lse / scale into every row of S, -Delta into every row of dP
            tc_mma_f16(tS, smem_desc_rows16(sAdd + YS * 2 * kAddBytes, kAddBytes),
                       smem_desc_rows16(sAdd + st * 2 * kAddBytes, kAddBytes), make_idesc(1, kX, 2 * kY), 0u);
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // S, dP
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              const uint64_t yk = y + i * (L::kYBytes >> 4) + (k / 4) * (kY * 128 >> 4) + 2 * (k % 4);
              if (kKeys)
                tc_mma_f16(tS + 64 * i, x + i * (L::kXBytes >> 4) + (k / 4) * (kX * 128 >> 4) + 2 * (k % 4), yk, idesc_s,
                           1u);
              else
                tc_mma_f16_ts(tS + 64 * i, tm + L::kXCol + DP / 2 * i + 8 * k, yk, idesc_s, k > 0 ? 1u : 0u);
            }
          }
          tc_commit(&s_full[bf]);
        }
      }
      const int u = t - (NB - 1);
      if (u >= 0) {
        const int st = u % YS, bf = u % NB;
        if (!(ok = mbar_wait_warp(&p_full[bf], (u / NB) & 1, abort_flag, status))) break;
        tc_fence_after();
        const uint32_t tP = tm + 128 * bf, tD = tP + 64;
        auto half = [](int k) { return 8 * k + (k < kY / 32 ? 0 : 16); };  // columns of P for query or key 16 k
        if (issuer) {
          const uint64_t d0 = smem_desc_sw128_mn(sY + st * L::kStage, kY * 128);
          const uint64_t d1 = d0 + (L::kYBytes >> 4);
#pragma unroll
          for (int k = 0; k < kY / 16; ++k)
            tc_mma_f16_ts(tm + L::kAcc, tD + half(k), d0 + (uint64_t)(2048 >> 4) * k, idesc_g, (u > 0 || k > 0) ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < kY / 16; ++k)
            tc_mma_f16_ts(tm + L::kAcc, tD + half(k) + 16, d0 + (uint64_t)(2048 >> 4) * k, idesc_g, 1u);
          if (kKeys) {
#pragma unroll
            for (int k = 0; k < kY / 16; ++k)
              tc_mma_f16_ts(tm + L::kAcc + DP, tP + half(k), d1 + (uint64_t)(2048 >> 4) * k, idesc_g,
                            (u > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit(&y_empty[st]);
        }
      }
    }
    if (issuer) {
      tc_commit(done);
      mbar_wait(done, 0, abort_flag, status);
    }
    __syncwarp();
  } else {
    // ---------------- P and dS, then the gradients out ----------------
    const int set = (warp - 2) >> 2, bf = set >> 1, h = set & 1, quarter = warp & 3;  // h: half of the columns
    const int r = x0 + quarter * 32 + lane;  // this thread's row of X: a key, or a query row
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + 128 * bf + lanes, tD = tS + 64;  // S and P, dP and dS
    const float c = w.scale * 1.4426950408889634f;
    const float2 c2 = make_float2(c, c);
    const int rlo = x0 + quarter * 32, rhi = rlo + 31;
    float2 nl = make_float2(0.f, 0.f), nd = nl;  // queries' side: the row's -lse and -Delta
    if (!kKeys) {
      const float* st = p.stat + (((int64_t)b * w.H + head0) * p.stat_tiles + r / kY) * 128 + r % kY;
      const bool have = r < p.stat_tiles * kY;
      nl.x = nl.y = have ? __ldg(st) : -INFINITY, nd.x = nd.y = have ? __ldg(st + 64) : 0.f;
    }
    bool ok = true;
    if (!kKeys && set < 2) {  // set 0 brings Q's rows into tensor memory, set 1 dO's
      const int64_t* step = set ? p.dout_step : p.q_step;
      const __nv_bfloat16* x = (set ? p.dout : p.q) + b * step[0] + r * step[1] + head0 * step[2];
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (r < w.Tq && 32 * c + 8 * u < w.D) v[u] = *reinterpret_cast<const uint4*>(x + 32 * c + 8 * u);
        }
        const uint32_t words[16] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w,
                                    v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
        tmem_st16(tmem + lanes + L::kXCol + DP / 2 * set + 16 * c, words);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x_full);
    }
    for (int t = bf; t < items; t += NB) {
      step_to(it, t, t == bf ? begin + bf : NB);
      const int y0 = it.y * kY;
      if (!(ok = mbar_wait_warp(&s_full[bf], (t / NB) & 1, abort_flag, status))) break;
      tc_fence_after();
      const int yc = y0 + 32 * h;
      const int qlo = kKeys ? w.offset + yc : w.offset + rlo, qhi = kKeys ? qlo + 31 : w.offset + rhi;
      const int klo = kKeys ? rlo : yc, khi = kKeys ? rhi : yc + 31;
      uint32_t pw[16], dw[16], lw[16];  // P, dS's upper part, and the rest of it
      const bool none = window_none(qlo, qhi, klo, khi, w.window, w.sinks);
      if (none) {
#pragma unroll
        for (int u = 0; u < 16; ++u) pw[u] = dw[u] = lw[u] = 0u;
      } else {
        uint32_t s[32], d[32];
        tmem_ld32_async(tS + 32 * h, s);
        tmem_ld32_async(tD + 32 * h, d);
        tmem_wait_ld_regs(s);
        tmem_wait_ld_regs(d);
        // visible pairs, bit by column; keys past the end of a padded sequence lie behind every query with a token
        uint32_t seen = 0xffffffffu;
        if (!window_all(qlo, qhi, klo, khi, w.window, w.sinks)) {
          seen = kKeys ? window_queries(qlo, r, w.window, w.sinks) : window_keys(w.offset + r, yc, w.window, w.sinks);
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const float2 s2 = make_float2(__uint_as_float(s[2 * u]), __uint_as_float(s[2 * u + 1]));
          const float2 d2 = make_float2(__uint_as_float(d[2 * u]), __uint_as_float(d[2 * u + 1]));
          const float2 x = kKeys ? __fmul2_rn(s2, c2) : __ffma2_rn(s2, c2, nl);
          const float2 pr = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          const float2 e = kKeys ? d2 : __fadd2_rn(d2, nd);
          const float2 ds = __fmul2_rn(pr, e);
          pw[u] = pack2<__nv_bfloat16>(pr.x, pr.y);
          const uint32_t dx = __float_as_uint(ds.x), dy = __float_as_uint(ds.y);
          dw[u] = __byte_perm(dx, dy, 0x7632);  // the upper halves: dS cut to bf16
          lw[u] = pack2<__nv_bfloat16>(ds.x - __uint_as_float(dx & 0xffff0000u), ds.y - __uint_as_float(dy & 0xffff0000u));
        }
        if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {  // clear what is hidden, whatever it came to
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const uint32_t two = seen >> (2 * u), keep = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
            pw[u] &= keep, dw[u] &= keep, lw[u] &= keep;
          }
        }
      }
      if (kKeys) tmem_st16(tS + 32 * h, pw);  // over the half of S, and of dP, that this warp has read
      tmem_st16(tD + 32 * h, dw);
      tmem_st16(tD + 32 * h + 16, lw);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[bf]);
    }
    if (ok && mbar_wait_warp(done, 0, abort_flag, status)) {
      tc_fence_after();
      const bool have = kKeys ? r < length : r < rows;
      // the gradients' 32-column chunks (keys' side: dK's, then dV's) go round the sets
#pragma unroll
      for (int k = 0; k < (kKeys ? 2 : 1) * (DP / 32); ++k) {
        if (k % L::kSets != set) continue;
        const bool first = k < DP / 32;
        const int h = first ? k : k - DP / 32;
        const float f = first ? w.scale : 1.f;
        __nv_bfloat16* g = first ? g0 : g1;
        const uint32_t tG = tmem + L::kAcc + lanes + (first ? 0 : DP);
        float o[32];
        tmem_read32(tG + 32 * h, o);
        if (slot >= 0) {
          float* out = p.partial + (((int64_t)slot * 2 + (first ? 0 : 1)) * kX + (r - x0)) * w.D + 32 * h;
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (32 * h + 4 * u < w.D)
              st_global_v4f(out + 4 * u, have ? o[4 * u] * f : 0.f, have ? o[4 * u + 1] * f : 0.f,
                            have ? o[4 * u + 2] * f : 0.f, have ? o[4 * u + 3] * f : 0.f);
        } else if (r < T) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (32 * h + 8 * u >= w.D) break;
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[k] = have ? pack2<__nv_bfloat16>(o[8 * u + 2 * k] * f, o[8 * u + 2 * k + 1] * f) : 0u;
            st_global_v4(grad_row(g, r) + 32 * h + 8 * u, x[0], x[1], x[2], x[3]);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Both sides in one launch, the keys' side first: its CTAs have the most work.
template <int DP>
__global__ void __launch_bounds__(WinBwd<DP>::kThreads, WinBwd<DP>::kCtas)
    window_backward_kernel(const __grid_constant__ WindowMaps m, const __grid_constant__ WindowGrad p, int key_ctas) {
  if ((int)blockIdx.x < key_ctas)
    window_side<DP, true>(m, p, blockIdx.x);
  else
    window_side<DP, false>(m, p, blockIdx.x - key_ctas);
}

// dK and dV of split key tiles: their partial sums added in order. One thread per four columns.
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WindowGrad p, int slots, int first_tile,
                                                          int tiles, int splits, int slot0) {
  const WindowParams& w = p.w;
  const int heads = w.H / w.group, b = blockIdx.z, kv = blockIdx.y, c = w.D / 4;
  const int64_t n = (int64_t)tiles * 2 * 128 * c;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int col = (int)(e % c) * 4, row = (int)(e / c % 128), which = (int)(e / (128 * c) % 2);
    const int tile = (int)(e / (2 * 128 * (int64_t)c));
    const int key = (first_tile + tile) * 128 + row;
    if (key >= w.Tk) continue;
    const int64_t slot = (int64_t)(b * heads + kv) * slots + slot0 + tile * splits;
    const float* src = p.partial + ((slot * 2 + which) * 128 + row) * w.D + col;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(src + (int64_t)s * 2 * 128 * w.D);
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    __nv_bfloat16* g = reinterpret_cast<__nv_bfloat16*>(which ? p.dv : p.dk) +
                       (((int64_t)b * w.Tk + key) * heads + kv) * w.D + col;
    *reinterpret_cast<uint2*>(g) = make_uint2(pack2<__nv_bfloat16>(t.x, t.y), pack2<__nv_bfloat16>(t.z, t.w));
  }
}

bool window_operand_ok(const void* ptr, const int64_t* stride, int B, int T, int heads);
int check_window(const NoiseWindow* a, bool token);
WindowParams window_params(const NoiseWindow* a, int* status);

struct WindowPlan {
  int q_tiles, k_tiles, sink_tiles, sink_splits, splits, slots;  // slots: partial sums per (sequence, key head)
  int64_t stat_bytes, add_bytes, bytes;
};

// How the keys' side is split: items (a 64-query tile of one head) per CTA at most `chunk`, the share that gives
// every SM two CTAs, but not less than 16, below which writing and joining the partial sums costs more than it
// saves. 148 SMs whatever the device, so that the workspace size is a function of the shape alone.
static WindowPlan window_plan(const NoiseWindow* a) {
  WindowPlan p{};
  p.q_tiles = (a->Tq + 63) / 64, p.k_tiles = (a->Tk + 127) / 128;
  const int64_t group = a->H / a->Hk;
  const int window = a->window < a->Tk ? a->window : a->Tk, sinks = a->sinks < a->Tk ? a->sinks : a->Tk;
  p.sink_tiles = (sinks + 127) / 128;
  const int64_t reach = min((int64_t)p.q_tiles, ((int64_t)window + 128) / 64 + 1);
  const int64_t plain = p.k_tiles - p.sink_tiles;
  const int64_t sink_items = group * p.q_tiles, items = group * reach;
  const int64_t total = (int64_t)a->B * a->Hk * (p.sink_tiles * sink_items + plain * items);
  const int64_t chunk = max((int64_t)16, (total + 2 * 148 - 1) / (2 * 148));
  // an uneven tile is only split when it would outlast an even one by more than half
  p.splits = plain > 0 && items > chunk + chunk / 2 ? (int)((items + chunk - 1) / chunk) : 1;
  const int64_t even = (items + p.splits - 1) / p.splits, sink_chunk = max(chunk, plain > 0 ? even : (int64_t)0);
  p.sink_splits = p.sink_tiles > 0 && sink_items > sink_chunk + sink_chunk / 2 ? (int)((sink_items + sink_chunk - 1) / sink_chunk) : 1;
  p.slots = (p.sink_splits > 1 ? p.sink_tiles * p.sink_splits : 0) + (p.splits > 1 ? (int)plain * p.splits : 0);
  p.stat_bytes = ((int64_t)a->B * a->H * p.q_tiles * 512 + 255) / 256 * 256;
  p.add_bytes = (int64_t)a->B * a->H * p.q_tiles * kAddBytes;
  p.bytes = p.stat_bytes + p.add_bytes + (int64_t)a->B * a->Hk * p.slots * 2 * 128 * a->D * 4;
  return p;
}

template <int DP>
static int launch_window_backward(const NoiseWindow* a, const void* dout, const int64_t* ds, WindowGrad& g,
                                  const WindowPlan& plan, cudaStream_t s) {
  using L = WinBwd<DP>;
  static KernelOptIn opt_in;
  if (!opt_in(window_backward_kernel<DP>, L::kSmem)) return kStatusLaunchFailed;
  WindowMaps m;
  auto map = [&](CUtensorMap* t, const void* ptr, int T, int heads, const int64_t* stride, int box) {
    return make_tmap_bthd(t, ptr, NOISE_BF16, a->B, T, heads, a->D, stride, (uint32_t)box);
  };
  if (map(&m.k128, a->k, a->Tk, a->Hk, a->k_stride, L::kX) || map(&m.v128, a->v, a->Tk, a->Hk, a->v_stride, L::kX) ||
      map(&m.q64, a->q, a->Tq, a->H, a->q_stride, L::kY) || map(&m.o64, dout, a->Tq, a->H, ds, L::kY) ||
      map(&m.k64, a->k, a->Tk, a->Hk, a->k_stride, L::kY) || map(&m.v64, a->v, a->Tk, a->Hk, a->v_stride, L::kY))
    return kStatusBadArgument;
  const int plain = plan.k_tiles - plan.sink_tiles;
  const int64_t group = a->H / a->Hk, places = plan.sink_tiles * plan.sink_splits + (int64_t)plain * plan.splits;
  const int64_t key_ctas = places * a->B * a->Hk, query_ctas = (int64_t)((a->Tq + 127) / 128) * a->B * a->H;
  if (key_ctas + query_ctas > INT32_MAX) return kStatusUnsupported;
  g.keys = tile_order((int)places, a->B * a->Hk, (int64_t)a->Tq * a->D * 4 * group);
  g.queries = tile_order((a->Tq + 127) / 128, a->B * a->H, (int64_t)a->Tk * a->D * 4 / group);
  LaunchScope scope(kKindAttention, s, 2 + (plan.sink_splits > 1) + (plan.splits > 1));
  window_stats_kernel<<<dim3(plan.q_tiles, a->H, a->B), 256, 0, s>>>(
      reinterpret_cast<const __nv_bfloat16*>(a->out), reinterpret_cast<const __nv_bfloat16*>(dout), a->B > 1 ? ds[0] : 0,
      a->Tq > 1 ? ds[1] : 0, a->H > 1 ? ds[2] : 0, g.w, const_cast<float*>(g.stat),
      const_cast<uint4*>(g.adds));
  window_backward_kernel<DP><<<(unsigned)(key_ctas + query_ctas), L::kThreads, L::kSmem, s>>>(m, g, (int)key_ctas);
  const int join = 64;
  if (plan.sink_splits > 1)
    window_join_kernel<<<dim3(min(join, plan.sink_tiles * a->D / 4), a->Hk, a->B), 256, 0, s>>>(
        g, plan.slots, 0, plan.sink_tiles, plan.sink_splits, 0);
  if (plan.splits > 1)
    window_join_kernel<<<dim3(min(join, plain * a->D / 4), a->Hk, a->B), 256, 0, s>>>(
        g, plan.slots, plan.sink_tiles, plain, plan.splits, plan.sink_splits > 1 ? plan.sink_tiles * plan.sink_splits : 0);
  return cudaGetLastError() == cudaSuccess ? kStatusOk : kStatusLaunchFailed;
}

}  // namespace noise

using namespace noise;

extern "C" int64_t noise_window_backward_workspace_bytes(const NoiseWindow* a) {
  if (!a || a->B < 0 || a->Tq < 1 || a->Tk < 1 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->D < 8 || a->D > 128 ||
      a->window < 0 || a->sinks < 0)
    return -1;
  return window_plan(a).bytes;
}

extern "C" int noise_window_attention_backward(const NoiseWindow* a, const void* dout, const int64_t* dout_stride,
                                               void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                               int* status, void* stream) {
  const int rc = check_window(a, false);
  if (rc != kStatusOk) return rc;
  // fp16 has no range for dS: products of probabilities far below 1 with gradients that are small already
  if (a->dtype != NOISE_BF16) return kStatusUnsupported;
  if (!status || !dq || !dk || !dv || !dout_stride || !is_aligned(dq, 16) || !is_aligned(dk, 16) || !is_aligned(dv, 16))
    return kStatusBadArgument;
  if (a->B == 0) return kStatusOk;
  if (!window_operand_ok(dout, dout_stride, a->B, a->Tq, a->H)) return kStatusBadArgument;
  const WindowPlan plan = window_plan(a);
  if (!workspace || !is_aligned(workspace, 16) || workspace_bytes < (size_t)plan.bytes) return kStatusWorkspaceTooSmall;
  WindowGrad g{};
  g.w = window_params(a, status);
  g.stat = reinterpret_cast<const float*>(workspace), g.stat_tiles = plan.q_tiles;
  uint8_t* at = reinterpret_cast<uint8_t*>(workspace) + plan.stat_bytes;
  g.adds = reinterpret_cast<const uint4*>(at), g.partial = reinterpret_cast<float*>(at + plan.add_bytes);
  g.dq = dq, g.dk = dk, g.dv = dv;
  g.q = reinterpret_cast<const __nv_bfloat16*>(a->q), g.dout = reinterpret_cast<const __nv_bfloat16*>(dout);
  const int64_t size[3] = {a->B, a->Tq, a->H};
  for (int i = 0; i < 3; ++i)
    g.q_step[i] = size[i] > 1 ? a->q_stride[i] : 0, g.dout_step[i] = size[i] > 1 ? dout_stride[i] : 0;
  g.sink_tiles = plan.sink_tiles, g.sink_splits = plan.sink_splits, g.splits = plan.splits, g.slots = plan.slots;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->D <= 64 ? launch_window_backward<64>(a, dout, dout_stride, g, plan, s)
                    : launch_window_backward<128>(a, dout, dout_stride, g, plan, s);
}
