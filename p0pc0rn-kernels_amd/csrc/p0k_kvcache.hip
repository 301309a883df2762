// p0k_kvcache.hip — writing K / V rows into the 8-bit cache and reading them back (layout: p0k_kv.h).
//
//   a block becomes whole: s = max |x| / 127 (1 where all are 0), code = x / s to the nearest, ties to even
//   read back: f16(code * s)
#include "p0k_device.h"
#include "p0k_kv.h"

namespace p0k {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
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

// One workgroup takes one block of one sequence and kv head, keys or values, and every thread 32 of its values, in
// registers from the first load to the last store. Keys: token tid / 4, d 16 c .. + 15 and 64 + 16 c .. (c = tid % 4): whole
// pieces of the cache. Values: tokens 4 (tid / 16) .. + 3, d 8 (tid % 16) .. + 7: the four tokens of a d are a word of a
// piece, and pieces are put together in LDS.
template <int KV>
struct Part {
  uint32_t tid;
  __device__ uint32_t tok(int i) const { return KV ? 4 * (tid >> 4) + i : tid >> 2; }                               // token and
  __device__ uint32_t d(int i) const { return KV ? 8 * (tid & 15) : 16 * (tid & 3) + (i >> 1) * 64 + (i & 1) * 8; }   // first d of x[i]
  // x from / to the tail, the values whose token passes `is`
  template <class F>
  __device__ void load_tail(const uint16_t *tail, u16x8 *x, F is) const {
    if constexpr (KV == 0) {
      if (is(tok(0))) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *(const u16x8 *)(tail + kv_ktail(tok(0), d(i)));
      }
    } else {
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; i++) any |= is(tok(i));
      if (!any) return;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const u16x4 w = *(const u16x4 *)(tail + kv_vtail(tok(0), d(0) + j));
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (is(tok(i))) x[i][j] = w[i];
      }
    }
  }
  template <class F>
  __device__ void store_tail(uint16_t *tail, const u16x8 *x, F is) const {
    if constexpr (KV == 0) {
      if (is(tok(0))) {
#pragma unroll
        for (int i = 0; i < 4; i++) *(u16x8 *)(tail + kv_ktail(tok(0), d(i))) = x[i];
      }
    } else {
      bool any = false, all = true;
#pragma unroll
      for (int i = 0; i < 4; i++) { any |= is(tok(i)); all &= is(tok(i)); }
      if (!any) return;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        uint16_t *at = tail + kv_vtail(tok(0), d(0) + j);
        if (all) {
          *(u16x4 *)at = (u16x4){x[0][j], x[1][j], x[2][j], x[3][j]};
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (is(tok(i))) at[i] = x[i][j];
        }
      }
    }
  }
};

template <int KV>
__device__ void append_block(const KvParams &p, const KvSeq &s, uint32_t blk, uint32_t k0, uint32_t end, uint32_t h, uint8_t *sC, float *sMax) {
  const uint32_t tid = threadIdx.x;
  const Part<KV> part{tid};
  const uint16_t *X = (KV ? p.V : p.K) + (KV ? p.vhs : p.khs) * h;
  const uint64_t rs = KV ? p.vrs : p.krs;
  u16x8 x[4];
  // the values of a block that this call brings
  auto fresh = [&](uint32_t block) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t t = block * KV_T + part.tok(i);
      if (t >= s.pos && t < end) {
        x[i] = *(const u16x8 *)(X + rs * (s.r0 + (t - s.pos)) + part.d(i));
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = kv_finite(x[i][j]);
      }
    }
  };
  auto keep = [&](uint32_t block) {              // and into the tail
    part.store_tail(p.tail + kv_tail_at(p, s.slot, block, h, KV), x, [&](uint32_t t) {
      const uint32_t tt = block * KV_T + t;
      return tt >= s.pos && tt < end;
    });
  };
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  fresh(blk);
  // The tail keeps the last block and the one before it. Of its two places, the first block's may still be read (the tokens
  // that it held before this call): that block's workgroup writes it, after it has read.
  const uint32_t last = end / KV_T;
  if (blk + 1 >= last && (blk == k0 || ((blk ^ k0) & 1))) keep(blk);
  if ((blk + 1) * KV_T <= end) {
    if (blk * KV_T < s.pos) {
      part.load_tail(p.tail + kv_tail_at(p, s.slot, blk, h, KV), x, [&](uint32_t t) { return blk * KV_T + t < s.pos; });
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = kv_finite(x[i][j]);   // (a tail that no call has written)
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
    uint8_t *codes = p.codes + kv_code_at(p, have ? page : 0u, h, KV);
    auto code = [&](uint16_t v) { return (uint32_t)(kv_code(h_val(v), sc, ri) + 128); };
    if constexpr (KV == 0) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        u32x4 w;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const u16x8 &v = x[2 * i + (g >> 1)];
          const int j = 4 * (g & 1);
          w[g] = code(v[j]) | code(v[j + 1]) << 8 | code(v[j + 2]) << 16 | code(v[j + 3]) << 24;
        }
        if (have) *(u32x4 *)(codes + kv_kcode(part.tok(0), part.d(2 * i))) = w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        *(uint32_t *)(sC + kv_vcode(part.tok(0), part.d(0) + j)) = code(x[0][j]) | code(x[1][j]) << 8 | code(x[2][j]) << 16 | code(x[3][j]) << 24;
      __syncthreads();
      if (have) {
#pragma unroll
        for (int i = 0; i < 2; i++) *(u32x4 *)(codes + 16 * (tid + 256 * i)) = *(const u32x4 *)(sC + 16 * (tid + 256 * i));
      }
    }
    if (have && tid == 0) p.scales[kv_scale_at(p, page, h, KV)] = sc;
  }
  if (blk == k0) {
    const uint32_t cb = ((last ^ k0) & 1) ? last - 1 : last;   // the one of the last two in the first block's place
    if (last >= 1 && cb > k0 && cb * KV_T < end) {
      __syncthreads();                           // (the whole workgroup has read the first block's tokens)
      fresh(cb);
      keep(cb);
    }
  }
}

__global__ __launch_bounds__(256) void k_kv_append(KvParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sC[KV_HEAD];
  __shared__ float sMax[4];
  const uint32_t item = blockIdx.x, h = blockIdx.y;
  const uint32_t b = kv_item_seq<KV_T>(p, item), base = kv_item_base<KV_T>(p, b);
  const KvSeq s = kv_seq(p, b);
  if (item < base || !s.ok || s.n == 0) return;
  const uint32_t cap = p.max_pages * KV_T, k0 = s.pos / KV_T, blk = k0 + (item - base);
  const uint32_t end = s.pos + s.n < cap ? s.pos + s.n : cap;
  if (blk >= p.max_pages || blk * KV_T >= end) return;
  if (blockIdx.z == 0) append_block<0>(p, s, blk, k0, end, h, sC, sMax);
  else append_block<1>(p, s, blk, k0, end, h, sC, sMax);
}

// code * scale of byte j of a word (byte = code + 128; 128 s is exact, so the fma rounds code * s once)
__device__ __forceinline__ uint16_t kv_value(uint32_t w, int j, float sc) {
  float v = fmaf((float)((w >> (8 * j)) & 255u), sc, -128.0f * sc);
  asm volatile("" : "+v"(v));                     // (rounded to fp32 before it is rounded to f16)
  return __builtin_bit_cast(uint16_t, (f16)v);
}

template <int KV>
__device__ void read_block(const KvParams &p, const KvSeq &s, uint32_t blk, uint32_t len, uint32_t h, uint8_t *sC) {
  const uint32_t tid = threadIdx.x, end = s.pos + s.n;
  const Part<KV> part{tid};
  u16x8 x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  const uint32_t page = blk < len / KV_T ? kv_page(p, s.slot, blk) : 0xffffffffu;
  if (blk == len / KV_T) {
    part.load_tail(p.tail + kv_tail_at(p, s.slot, blk, h, KV), x, [&](uint32_t t) { return blk * KV_T + t < len; });
  } else if (page != 0xffffffffu) {
    const uint8_t *codes = p.codes + kv_code_at(p, page, h, KV);
    const float sc = p.scales[kv_scale_at(p, page, h, KV)];
    if constexpr (KV == 0) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const u32x4 w = *(const u32x4 *)(codes + kv_kcode(part.tok(0), part.d(2 * i)));
#pragma unroll
        for (int j = 0; j < 16; j++) x[2 * i + (j >> 3)][j & 7] = kv_value(w[j >> 2], j & 3, sc);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) *(u32x4 *)(sC + 16 * (tid + 256 * i)) = *(const u32x4 *)(codes + 16 * (tid + 256 * i));
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t w = *(const uint32_t *)(sC + kv_vcode(part.tok(0), part.d(0) + j));
#pragma unroll
        for (int i = 0; i < 4; i++) x[i][j] = kv_value(w, i, sc);
      }
    }
  }
  uint16_t *Y = (KV ? p.Vo : p.Ko) + (KV ? p.vhs : p.khs) * h;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t t = blk * KV_T + part.tok(i);
    if (t >= s.pos && t < end) *(u16x8 *)(Y + (KV ? p.vrs : p.krs) * (s.r0 + (t - s.pos)) + part.d(i)) = x[i];
  }
}

__global__ __launch_bounds__(256) void k_kv_read(KvParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sC[KV_HEAD];
  const uint32_t item = blockIdx.x, h = blockIdx.y;
  const uint32_t b = kv_item_seq<KV_T>(p, item), base = kv_item_base<KV_T>(p, b);
  const KvSeq s = kv_seq(p, b);
  if (item < base || s.n == 0) return;
  const uint32_t blk = s.pos / KV_T + (item - base);
  if (blk * KV_T >= s.pos + s.n) return;
  const int32_t held = p.len[b];
  const uint32_t cap = p.max_pages * KV_T, len = !s.ok || held < 0 ? 0u : (uint32_t)held < cap ? (uint32_t)held : cap;
  if (blockIdx.z == 0) read_block<0>(p, s, blk, len, h, sC);
  else read_block<1>(p, s, blk, len, h, sC);
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
