// What the kernels of the sliding-window attention with sinks share: parameters, the visibility of a
// block of scores, the walk over a query tile's key tiles, and tensor maps of [B, T, heads, D] operands.
#pragma once

#include "operators.cuh"
#include "ptx.cuh"

namespace noise {

struct WindowParams {
  int B, Tq, Tk, H, group, D, offset, window, sinks;
  float scale;
  const int* lengths;  // [B] or null
  void* out;           // [B, Tq, H, D]
  float* lse;          // [B, H, Tq]
  int* status;
};

// Tokens of sequence b that a query can see or be: those before its length and up to the last query. What lies behind, such
// as the free rows of a cache, is padding whatever it holds.
__device__ __forceinline__ int window_length(const WindowParams& p, int b) {
  const int end = p.offset + p.Tq;
  return p.lengths ? min(max(__ldg(p.lengths + b), 0), end) : end;
}

// Queries qlo .. qhi against keys klo .. khi: no pair visible, or every pair.
__device__ __forceinline__ bool window_none(int qlo, int qhi, int klo, int khi, int window, int sinks) {
  return klo > qhi || (qlo - khi > window && klo >= sinks);
}
__device__ __forceinline__ bool window_all(int qlo, int qhi, int klo, int khi, int window, int sinks) {
  return khi <= qlo && (qhi - klo <= window || khi < sinks);
}

// The low n bits (n clamped to [0, 32]).
__device__ __forceinline__ uint32_t low_bits(int n) {
  uint32_t r;
  asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(r) : "r"(max(n, 0)));
  return r;
}

// Bit u: query q sees key k0 + u (u < 32).
__device__ __forceinline__ uint32_t window_keys(int q, int k0, int window, int sinks) {
  return low_bits(q - k0 + 1) & (~low_bits(q - window - k0) | low_bits(sinks - k0));
}

// Bit u: query q0 + u sees key k (u < 32).
__device__ __forceinline__ uint32_t window_queries(int q0, int k, int window, int sinks) {
  return ~low_bits(k - q0) & (k < sinks ? 0xffffffffu : low_bits(k + window - q0 + 1));
}

// 32 columns of this warp's tensor memory lanes; the wait names the registers, so that no use moves before it.
__device__ __forceinline__ void tmem_read32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld32_async(taddr, r);
  tmem_wait_ld_regs(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// The order in which CTAs take (tile, sequence and head) pairs: heavy tiles first, over groups of pairs whose
// streamed operands fit the L2 cache together, so that the last CTAs to run are short ones.
struct TileOrder {
  int tiles, pairs, group;  // pairs: sequences x heads
  __device__ __forceinline__ void at(int index, int& tile, int& pair) const {
    const int full = tiles * group, g = index / full, rest = index - g * full;
    const int size = min(group, pairs - g * group);
    tile = rest / size;
    pair = g * group + rest - tile * size;
  }
};

inline TileOrder tile_order(int tiles, int pairs, int64_t bytes_per_pair) {
  const int64_t fit = (64ll << 20) / (bytes_per_pair > 0 ? bytes_per_pair : 1);
  return TileOrder{tiles, pairs, (int)(fit < 1 ? 1 : fit < pairs ? fit : pairs)};
}

int make_tmap_bthd(CUtensorMap* map, const void* ptr, int dtype, int B, int T, int heads, int D, const int64_t* stride,
                   uint32_t box_rows);
int device_sm_count();

}  // namespace noise
