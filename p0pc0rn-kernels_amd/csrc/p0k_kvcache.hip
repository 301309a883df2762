// p0k_kvcache.hip — writing K / V rows into the 8-bit cache and reading them back (layout: p0k_kv.h).
//
//   a block becomes whole: s = max |x| / 127 (1 where all are 0), code = x / s to the nearest, ties to even
//   read back: f16(code * s)
#include "p0k_device.h"
#include "p0k_kv.h"

namespace p0k {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// f16 bits held to the finite range, NaN to 0
__device__ __forceinline__ uint16_t kv_finite(uint16_t x) {
  const uint16_t m = x & 0x7fffu;
  return m > 0x7c00u ? (uint16_t)0 : m == 0x7c00u ? (uint16_t)(x - 1) : x;
}
// x / s rounded to the nearest integer, ties to even, exactly: the estimate is off by less than one, and x - c s is exact
// in one fma where it is near s / 2 (x has 11 bits and is at least s / 2 there; the difference needs no more than 24)
__device__ __forceinline__ int kv_code(float x, float s, float rs) {
  float c = __builtin_rintf(x * rs);
  const float r = fmaf(-c, s, x), h = 0.5f * s;
  const bool odd = ((int)c & 1) != 0;
  if (r > h || (r == h && odd)) c += 1.0f;
  else if (r < -h || (r == -h && odd)) c -= 1.0f;
  return (int)c;
}

// One workgroup takes one block of one sequence and kv head, keys or values: thread (t, c) holds d 16 c .. + 15 and 64 + 16 c
// .. + 15 of token t, its 32 values in registers, so a row is read once.
__global__ __launch_bounds__(256) void k_kv_append(KvParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sC[KV_T][KV_D + 4];
  __shared__ float sMax[4];
  const uint32_t item = blockIdx.x, h = blockIdx.y, kv = blockIdx.z, tid = threadIdx.x;
  const uint32_t b = kv_item_seq<KV_T>(p, item), base = kv_item_base<KV_T>(p, b);
  const KvSeq s = kv_seq(p, b);
  if (item < base || !s.ok || s.n == 0) return;
  const uint32_t cap = p.max_pages * KV_T, k0 = s.pos / KV_T, blk = k0 + (item - base);
  const uint32_t end = s.pos + s.n < cap ? s.pos + s.n : cap;
  if (blk >= p.max_pages || blk * KV_T >= end) return;

  const uint16_t *X = (kv ? p.V : p.K) + (kv ? p.vhs : p.khs) * h;
  const uint64_t rs = kv ? p.vrs : p.krs;
  const uint32_t t = tid >> 2, c = tid & 3;
  u16x8 x[4];                                    // d 16 c, 16 c + 8, 64 + 16 c, 72 + 16 c of token t
  auto dof = [&](int i) { return 16 * c + (i >> 1) * 64 + (i & 1) * 8; };
  // the rows of a block that this call brings (true: token t is one)
  auto fresh = [&](uint32_t block) {
    const uint32_t tok = block * KV_T + t;
    const bool is = tok >= s.pos && tok < end;
    if (is) {
      const uint16_t *row = X + rs * (s.r0 + (tok - s.pos));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = *(const u16x8 *)(row + dof(i));
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = kv_finite(x[i][j]);
      }
    }
    return is;
  };
  auto keep = [&](uint32_t block) {              // token t's values into the tail
    uint16_t *tail = p.tail + kv_tail_at(p, s.slot, block, h, kv);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (kv == 0) {
        *(u16x8 *)(tail + kv_ktail(t, dof(i))) = x[i];
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) tail[kv_vtail(t, dof(i) + j)] = x[i][j];
      }
    }
  };
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  const bool is = fresh(blk), whole = (blk + 1) * KV_T <= end;
  // The tail keeps the last block and the one before it. Of its two places, the first block's may still be read (the tokens
  // that it held before this call): that block's workgroup writes it, after it has read.
  const uint32_t last = end / KV_T;
  if (is && blk + 1 >= last && (blk == k0 || ((blk ^ k0) & 1))) keep(blk);
  if (whole) {
    const uint32_t tok = blk * KV_T + t;
    if (tok < s.pos) {
      const uint16_t *tail = p.tail + kv_tail_at(p, s.slot, blk, h, kv);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (kv == 0) {
          x[i] = *(const u16x8 *)(tail + kv_ktail(t, dof(i)));
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[i][j] = tail[kv_vtail(t, dof(i) + j)];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = kv_finite(x[i][j]);   // (a tail that no call has written)
      }
    }
    uint32_t mx = 0;                             // |x| as bits: finite f16 order as integers
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) mx = max(mx, (uint32_t)(x[i][j] & 0x7fffu));
    for (int o = 32; o; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    if ((tid & 63) == 0) sMax[tid >> 6] = h_val((uint16_t)mx);
    __syncthreads();
    const float amax = fmaxf(fmaxf(sMax[0], sMax[1]), fmaxf(sMax[2], sMax[3]));
    const float sc = amax > 0.0f ? amax / 127.0f : 1.0f, ri = 1.0f / sc;
    const uint32_t page = kv_page(p, s.slot, blk);
    const bool have = page != 0xffffffffu;
    uint8_t *codes = p.codes + kv_code_at(p, have ? page : 0u, h, kv);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int g = 0; g < 2; g++) {
        uint32_t v = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) v |= (uint32_t)(kv_code(h_val(x[i][4 * g + j]), sc, ri) + 128) << (8 * j);
        w[2 * i + g] = v;
      }
    if (kv == 0) {
      if (have) {
#pragma unroll
        for (int i = 0; i < 2; i++)
          *(u32x4 *)(codes + kv_kcode(t, 64 * i + 16 * c)) = (u32x4){w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) *(uint32_t *)&sC[t][16 * c + (i >> 2) * 64 + (i & 3) * 4] = w[i];
      __syncthreads();
      if (have) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const uint32_t pc = tid + 256 * i, tq = 32 * (pc >> 8) + 4 * ((pc >> 4) & 3), d = 32 * ((pc >> 6) & 3) + (pc & 15);
          u32x4 o;
#pragma unroll
          for (int g = 0; g < 4; g++) {          // bytes 4 g ..: d + 16 (g / 2), tokens tq + 16 (g % 2) ..
            uint32_t v = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) v |= (uint32_t)sC[tq + 16 * (g & 1) + j][d + 16 * (g >> 1)] << (8 * j);
            o[g] = v;
          }
          *(u32x4 *)(codes + 16 * pc) = o;
        }
      }
    }
    if (have && tid == 0) p.scales[kv_scale_at(p, page, h, kv)] = sc;
  }
  if (blk == k0) {
    const uint32_t cb = ((last ^ k0) & 1) ? last - 1 : last;   // the one of the last two in the first block's place
    if (cb > k0 && cb * KV_T < end && last >= 1) {
      __syncthreads();                           // (the whole workgroup has read the first block's tokens)
      if (fresh(cb)) keep(cb);
    }
  }
}

__global__ __launch_bounds__(256) void k_kv_read(KvParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sC[KV_T][KV_D + 4];
  const uint32_t item = blockIdx.x, h = blockIdx.y, kv = blockIdx.z, tid = threadIdx.x;
  const uint32_t b = kv_item_seq<KV_T>(p, item), base = kv_item_base<KV_T>(p, b);
  const KvSeq s = kv_seq(p, b);
  if (item < base || s.n == 0) return;
  const uint32_t blk = s.pos / KV_T + (item - base), t = tid >> 2, c = tid & 3, end = s.pos + s.n;
  if (blk * KV_T >= end) return;
  const int32_t held = p.len[b];
  const uint32_t cap = p.max_pages * KV_T, len = !s.ok || held < 0 ? 0u : (uint32_t)held < cap ? (uint32_t)held : cap;
  const uint32_t tok = blk * KV_T + t;
  const bool open = blk == len / KV_T;
  const uint32_t page = open || blk > len / KV_T ? 0xffffffffu : kv_page(p, s.slot, blk);
  u16x8 x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  auto dof = [&](int i) { return 16 * c + (i >> 1) * 64 + (i & 1) * 8; };
  if (open) {
    if (tok < len) {
      const uint16_t *tail = p.tail + kv_tail_at(p, s.slot, blk, h, kv);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (kv == 0) {
          x[i] = *(const u16x8 *)(tail + kv_ktail(t, dof(i)));
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[i][j] = tail[kv_vtail(t, dof(i) + j)];
        }
      }
    }
  } else if (page != 0xffffffffu) {
    const uint8_t *codes = p.codes + kv_code_at(p, page, h, kv);
    const float sc = p.scales[kv_scale_at(p, page, h, kv)];
    u32x4 w[2];
    if (kv == 0) {
#pragma unroll
      for (int i = 0; i < 2; i++) w[i] = *(const u32x4 *)(codes + kv_kcode(t, 64 * i + 16 * c));
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t pc = tid + 256 * i, tq = 32 * (pc >> 8) + 4 * ((pc >> 4) & 3), d = 32 * ((pc >> 6) & 3) + (pc & 15);
        const u32x4 o = *(const u32x4 *)(codes + 16 * pc);
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
          for (int j = 0; j < 4; j++) sC[tq + 16 * (g & 1) + j][d + 16 * (g >> 1)] = (uint8_t)(o[g] >> (8 * j));
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) w[i][j] = *(const uint32_t *)&sC[t][64 * i + 16 * c + 4 * j];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = ((float)((w[i >> 1][2 * (i & 1) + (j >> 2)] >> (8 * (j & 3))) & 255u) - 128.0f) * sc;
        x[i][j] = __builtin_bit_cast(uint16_t, (f16)v);
      }
  }
  if (tok >= s.pos && tok < end) {
    uint16_t *row = (kv ? p.Vo : p.Ko) + (kv ? p.vhs : p.khs) * h + (kv ? p.vrs : p.krs) * (s.r0 + (tok - s.pos));
#pragma unroll
    for (int i = 0; i < 4; i++) *(u16x8 *)(row + dof(i)) = x[i];
  }
}

hipError_t launch_kv_append(const KvParams &p, hipStream_t s) {
  if (p.rows == 0 || p.B == 0 || p.Hkv == 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv_append, dim3(p.rows / KV_T + 2 * p.B, p.Hkv, 2), dim3(256), 0, s, p);
  return hipGetLastError();
}
hipError_t launch_kv_read(const KvParams &p, hipStream_t s) {
  if (p.rows == 0 || p.B == 0 || p.Hkv == 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv_read, dim3(p.rows / KV_T + 2 * p.B, p.Hkv, 2), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace p0k
