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

// Valid tokens of sequence b, within [0, Tk].
__device__ __forceinline__ int window_length(const WindowParams& p, int b) {
  return p.lengths ? min(max(__ldg(p.lengths + b), 0), p.Tk) : p.Tk;
}

// Query at position q sees key k.
__device__ __forceinline__ bool window_sees(int q, int k, int window, int sinks) {
  return k <= q && (q - k <= window || k < sinks);
}

// Queries qlo .. qhi against keys klo .. khi: no pair visible, or every pair.
__device__ __forceinline__ bool window_none(int qlo, int qhi, int klo, int khi, int window, int sinks) {
  return klo > qhi || (qlo - khi > window && klo >= sinks);
}
__device__ __forceinline__ bool window_all(int qlo, int qhi, int klo, int khi, int window, int sinks) {
  return khi <= qlo && (qhi - klo <= window || khi < sinks);
}

// 32 columns of this warp's tensor memory lanes; the wait names the registers, so that no use moves before it.
__device__ __forceinline__ void tmem_read32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ld32_async(taddr, r);
  tmem_wait_ld_regs(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

int make_tmap_bthd(CUtensorMap* map, const void* ptr, int dtype, int B, int T, int heads, int D, const int64_t* stride,
                   uint32_t box_rows);
int device_sm_count();

}  // namespace noise
