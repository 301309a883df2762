// p0k_rope.hip — rotary positions over rows of heads (size 128, f16): interleaved or half pairs, the first rd values of a
// head, any frequencies.
//
//   y1 = m (x1 cos a - x2 sin a), y2 = m (x2 cos a + x1 sin a),  a = t f_i of the row's token t
//
// An angle is a fraction of a turn: f_i / 2 pi comes as a 64-bit fixed-point fraction from the host, and t times it wraps
// by itself, so the error does not grow with t (fp32 angles are off by 0.06 rad at t = 10^6).
#include "p0k_device.h"
#include "p0k_kv.h"

namespace p0k {

// Sixteen threads share a row, eight values of a head each; a thread computes its sines and cosines once and walks the heads
// of its group with them. A pair's two values lie in one thread (interleaved) or in two of the same wave, whose loads come
// before its stores: x may be y.
__global__ __launch_bounds__(256) void k_rope(RopeParams p, uint32_t hg) {
  __shared__ uint64_t turn[64];
  if (threadIdx.x < 64) turn[threadIdx.x] = p.turn[threadIdx.x];
  __syncthreads();
  const uint32_t r = blockIdx.x * 16 + (threadIdx.x >> 4), c = threadIdx.x & 15, rot = p.rd >> 1;
  if (r >= p.rows) return;
  int64_t t;
  if (p.cu) {
    // the sequence of the row: the largest b with cu[b] <= r
    uint32_t lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (kv_row0(p.cu, mid, p.rows) <= r) lo = mid;
      else hi = mid;
    }
    const uint32_t r0 = kv_row0(p.cu, lo, p.rows);
    if (r < r0 || r >= kv_row0(p.cu, lo + 1, p.rows)) return;
    t = (int64_t)p.pos[lo] + (r - r0);
  } else {
    t = p.pos[r];
  }
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t d = 8 * c + j, i = p.half ? (d < rot ? d : d - rot) : d >> 1;
    cs[j] = 1.0f;
    sn[j] = 0.0f;
    if (d < p.rd) {
      const int32_t a = (int32_t)(((uint64_t)t * turn[i]) >> 32);                  // the fraction's upper half, signed
      float s, o;
      sincospif((float)a * 0x1p-31f, &s, &o);
      cs[j] = o * p.mscale;
      sn[j] = (p.half ? d < rot : (d & 1) == 0) ? -s * p.mscale : s * p.mscale;   // y[d] = cs x[d] + sn x[its partner]
    }
  }
  const uint32_t h0 = blockIdx.y * hg, h1 = h0 + hg < p.H ? h0 + hg : p.H;
  for (uint32_t h = h0; h < h1; h++) {
    const uint16_t *x = p.X + p.xrs * r + p.xhs * h;
    const f16x8 v = *(const f16x8 *)(x + 8 * c);
    f16x8 o = v;
    if (8 * c < p.rd) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t d = 8 * c + j;
        if (d < p.rd) o[j] = __builtin_bit_cast(f16, x[p.half ? (d < rot ? d + rot : d - rot) : d ^ 1u]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++)
        o[j] = 8 * c + j < p.rd ? (f16)((float)v[j] * cs[j] + (float)o[j] * sn[j]) : v[j];
    }
    *(f16x8 *)(p.Y + p.yrs * r + p.yhs * h + 8 * c) = o;
  }
}

hipError_t launch_rope(const RopeParams &p, hipStream_t s) {
  if (p.rows == 0 || p.H == 0) return hipSuccess;
  hipLaunchKernelGGL(k_rope, dim3((p.rows + 15) / 16, p.H), dim3(256), 0, s, p, 1u);
  return hipGetLastError();
}

}  // namespace p0k
