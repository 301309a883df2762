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

// How a value's partner is reached: in the same thread (interleaved pairs), in another thread's 16 bytes (halves of a multiple
// of 8 values), one by one (other halves)
enum { R_PAIRS = 0, R_HALF8 = 1, R_HALF = 2 };

// Sixteen threads share a row, eight values of a head each; a thread computes its sines and cosines once and walks the heads
// of its group with them, four heads' loads in flight. A partner in another thread is one of the same wave, whose loads come
// before its stores: x may be y. HBM-bound: 4001 rows of 40 heads (82 MB) 15.2 us, 5.4 TB/s (33.4 with a head per workgroup and a
// load per partner); 16 rows 4.8 us, back to back in a graph: a launch, then the search of the row's sequence, its position and the
// angles one after another (the host's part of a call, the frequencies, takes 1.8 us beside it).
template <int MODE>
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
    const uint32_t d = 8 * c + j, i = MODE != R_PAIRS ? (d < rot ? d : d - rot) : d >> 1;
    cs[j] = 1.0f;
    sn[j] = 0.0f;
    if (d < p.rd) {
      const int32_t a = (int32_t)(((uint64_t)t * turn[i]) >> 32);                  // the fraction's upper half, signed
      float s, o;
      sincospif((float)a * 0x1p-31f, &s, &o);
      cs[j] = o * p.mscale;
      sn[j] = (MODE != R_PAIRS ? d < rot : (d & 1) == 0) ? -s * p.mscale : s * p.mscale;   // y[d] = cs x[d] + sn x[its partner]
    }
  }
  const uint32_t h0 = blockIdx.y * hg, h1 = h0 + hg < p.H ? h0 + hg : p.H;
  const bool turns = 8 * c < p.rd;
  const uint16_t *x = p.X + p.xrs * r + 8 * c;
  uint16_t *y = p.Y + p.yrs * r + 8 * c;
  const int32_t to = MODE == R_HALF8 ? (8 * c < rot ? (int32_t)rot : -(int32_t)rot) : 0;
  for (uint32_t h = h0; h < h1; h += 4) {
    f16x8 v[4], o[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
      const uint16_t *xh = x + p.xhs * (h + i < h1 ? h + i : h1 - 1);
      v[i] = *(const f16x8 *)xh;
      o[i] = v[i];
      if (MODE == R_HALF8 && turns) o[i] = *(const f16x8 *)(xh + to);
      if (MODE == R_HALF && turns) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t d = 8 * c + j;
          if (d < p.rd) o[i][j] = __builtin_bit_cast(f16, xh[j + (d < rot ? (int32_t)rot : -(int32_t)rot)]);
        }
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
      if (h + i >= h1) break;
      if (turns) {
        const f16x8 w = v[i], q = MODE == R_PAIRS ? (f16x8){w[1], w[0], w[3], w[2], w[5], w[4], w[7], w[6]} : o[i];
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = 8 * c + j < p.rd ? (f16)((float)w[j] * cs[j] + (float)q[j] * sn[j]) : w[j];
      }
      *(f16x8 *)(y + p.yhs * (h + i)) = v[i];
    }
  }
}

// Heads a thread walks: all of them where the rows alone fill the GPU (2048 workgroups), else as few as do
hipError_t launch_rope(const RopeParams &p, hipStream_t s) {
  if (p.rows == 0 || p.H == 0 || (p.cu && p.B == 0)) return hipSuccess;
  const uint32_t wgs = (p.rows + 15) / 16, groups = wgs >= 2048 ? 1 : (2048 + wgs - 1) / wgs;
  uint32_t hg = (p.H + groups - 1) / groups;
  hg = hg < 4 ? 4 : (hg + 3) / 4 * 4;
  const dim3 grid(wgs, (p.H + hg - 1) / hg), block(256);
  if (!p.half) hipLaunchKernelGGL(k_rope<R_PAIRS>, grid, block, 0, s, p, hg);
  else if (p.rd % 16 == 0) hipLaunchKernelGGL(k_rope<R_HALF8>, grid, block, 0, s, p, hg);
  else hipLaunchKernelGGL(k_rope<R_HALF>, grid, block, 0, s, p, hg);
  return hipGetLastError();
}

}  // namespace p0k
