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
// the low bytes of four words
__device__ __forceinline__ uint32_t kv_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return perm(perm(d, c, 0x0c0c0400u), perm(b, a, 0x0c0c0400u), 0x05040100u);
}
// The bytes (code + 128) of a thread's 32 values, eight words of four: of consecutive d (keys) or of the four tokens of a d
// (values). x / s is estimated as x rs, off by less than 2^-16 (127 x 2^-24 of rs and 2^-18 of the product), and the sum with
// 2^23 + 128 rounds it to the nearest integer. Where an estimate of the wave lies within that of a border, all of them are
// settled exactly: x - c s takes no rounding where it is near s / 2 (x has 11 bits and is at least s / 2 there, the difference
// needs no more than 24), and ties go to the even code.
template <int KV>
__device__ __forceinline__ void kv_codes(const u16x8 *x, float s, uint32_t *w) {
  const float rs = 1.0f / s, big = 8388608.0f + 128.0f;
  auto val = [&](int g, int j) { return h_val(KV ? x[j][g] : x[g >> 1][4 * (g & 1) + j]); };
  float far = 0.0f;
#pragma unroll
  for (int g = 0; g < 8; g++) {
    float z[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float y = val(g, j) * rs;
      z[j] = y + big;
      far = fmaxf(far, fabsf(y - (z[j] - big)));
    }
    w[g] = kv_bytes(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
  }
  if (__any(far > 0.5f - 0x1p-16f)) {
    const float h = 0.5f * s;
#pragma unroll
    for (int g = 0; g < 8; g++) {
      uint32_t z[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int c = (int)((w[g] >> (8 * j)) & 255u) - 128;
        const float r = fmaf(-(float)c, s, val(g, j));
        const bool odd = (c & 1) != 0;
        z[j] = (uint32_t)(c + 128 + (r > h || (r == h && odd) ? 1 : r < -h || (r == -h && odd) ? -1 : 0));
      }
      w[g] = kv_bytes(z[0], z[1], z[2], z[3]);
    }
  }
}
// the largest |x| of a thread's values, as f16 bits (finite numbers order as integers; above: infinities, NaN)
__device__ __forceinline__ uint32_t kv_amax(const u16x8 *x) {
  const u16x8 m = {0x7fff, 0x7fff, 0x7fff, 0x7fff, 0x7fff, 0x7fff, 0x7fff, 0x7fff};
  const u16x8 a = __builtin_elementwise_max(__builtin_elementwise_max(x[0] & m, x[1] & m), __builtin_elementwise_max(x[2] & m, x[3] & m));
  uint32_t r = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) r = max(r, (uint32_t)a[j]);
  return r;
}
__device__ __forceinline__ void kv_hold(u16x8 *x) {       // infinities to the largest value, NaN to 0
  if (kv_amax(x) < 0x7c00u) return;
#pragma unroll
  for (int i = 0; i < 32; i++) x[i >> 3][i & 7] = kv_finite(x[i >> 3][i & 7]);
}

// One workgroup takes one block of one sequence and kv head, keys or values, and every thread 32 of its values, in
// registers from the first load to the last store. Keys: token tid / 4, d 16 c .. + 15 and 64 + 16 c .. (c = tid % 4): whole
// pieces of the cache. Values: tokens 4 (tid / 16) .. + 3, d 8 (tid % 16) .. + 7: the four tokens of a d are a word of a
// piece, and pieces are put together in LDS.
// 5000 rows of 8 heads: append 12.9 us (31 MB, 2.4 TB/s: the loads of all workgroups, then 5.5 us of VALU), read 9.0; 16384
// rows read back 23.0 us (100 MB, 4.4 TB/s). One token of 64 sequences: append 5.7 us (5.0 without `held`, whose entries come from
// memory with the rows).
template <int KV>
struct Part {
  uint32_t tid;
  __device__ uint32_t tok(int i) const { return KV ? 4 * (tid >> 4) + i : tid >> 2; }                               // token and
  __device__ uint32_t d(int i) const { return KV ? 8 * (tid & 15) : 16 * (tid & 3) + (i >> 1) * 64 + (i & 1) * 8; }   // first d of x[i]
  // x from / to the tail, the values whose token passes `is` (load: by the whole workgroup; a piece of values holds eight
  // tokens of a d, so they go through LDS, 16 KB as [four tokens][d])
  template <class F>
  __device__ void load_tail(const uint16_t *tail, u16x8 *x, uint8_t *lds, F is) const {
    if constexpr (KV == 0) {
      if (is(tok(0))) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *(const u16x8 *)(tail + kv_ktail(tok(0), d(i)));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t pc = tid + 256 * i, g = 8 * (pc >> 9) + ((pc >> 4) & 3), dd = 16 * ((pc >> 6) & 7) + (pc & 15);
        const u32x4 w = *(const u32x4 *)(tail + 8 * pc);
        *(u32x2 *)(lds + (g * KV_D + dd) * 8) = (u32x2){w.x, w.y};
        *(u32x2 *)(lds + ((g + 4) * KV_D + dd) * 8) = (u32x2){w.z, w.w};
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const u16x4 w = *(const u16x4 *)(lds + ((tid >> 4) * KV_D + d(0) + j) * 8);
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

// A head's codes in LDS: runs of 16 pieces (256 bytes: all banks), each moved on by a piece, since the words that a wave writes or
// reads at once lie at the same places of 16 runs
__device__ __forceinline__ uint32_t kv_lds(uint32_t code) { return code + (code >> 8) * 16; }

// code * scale of byte j of a word (byte = code + 128; 128 s is exact, so the fma rounds code * s once)
__device__ __forceinline__ uint16_t kv_value(uint32_t w, int j, float sc) {
  float v = fmaf((float)((w >> (8 * j)) & 255u), sc, -128.0f * sc);
  asm volatile("" : "+v"(v));                     // (rounded to fp32 before it is rounded to f16)
  return __builtin_bit_cast(uint16_t, (f16)v);
}

// a block's values x from its codes, as f16, those whose token passes `is` (by the whole workgroup; values go through LDS)
template <int KV, class F>
__device__ __forceinline__ void load_codes(const KvParams &p, const Part<KV> &part, uint32_t page, uint32_t h, u16x8 *x, uint8_t *sC, F is) {
  const uint8_t *codes = p.codes + kv_code_at(p, page, h, KV);
  const float sc = p.scales[kv_scale_at(p, page, h, KV)];
  if constexpr (KV == 0) {
    if (!is(part.tok(0))) return;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const u32x4 w = *(const u32x4 *)(codes + kv_kcode(part.tok(0), part.d(2 * i)));
#pragma unroll
      for (int j = 0; j < 16; j++) x[2 * i + (j >> 3)][j & 7] = kv_value(w[j >> 2], j & 3, sc);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) *(u32x4 *)(sC + kv_lds(16 * (part.tid + 256 * i))) = *(const u32x4 *)(codes + 16 * (part.tid + 256 * i));
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t w = *(const uint32_t *)(sC + kv_lds(kv_vcode(part.tok(0), part.d(0) + j)));
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (is(part.tok(i))) x[i][j] = kv_value(w, i, sc);
    }
  }
}

template <int KV>
__device__ void append_block(const KvParams &p, const KvSeq &s, uint32_t blk, uint32_t k0, uint32_t end, uint32_t h, uint8_t *sC, float *sMax) {
  const uint32_t tid = threadIdx.x;
  const Part<KV> part{tid};
  const uint16_t *X = (KV ? p.V : p.K) + (KV ? p.vhs : p.khs) * h;
  const uint64_t rs = KV ? p.vrs : p.krs;
  const int32_t entry = p.table[(uint64_t)s.slot * p.max_pages + blk];   // (asked for before it is needed)
  auto page_of = [&] { return entry >= 0 && (uint32_t)entry < p.pages ? (uint32_t)entry : 0xffffffffu; };
  const bool inside = blk * KV_T < s.pos;
  int32_t *held = p.held && blk == k0 ? kv_held(p, s.slot, h, KV) : nullptr;
  const int32_t places = held ? held[tid & 1] : 0;
  u16x8 x[4];
  // the values of a block that this call brings
  auto fresh = [&](uint32_t block) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t t = block * KV_T + part.tok(i);
      if (t >= s.pos && t < end) x[i] = *(const u16x8 *)(X + rs * (s.r0 + (t - s.pos)) + part.d(i));
    }
    kv_hold(x);
  };
  auto keep = [&](uint32_t block, uint32_t from, uint32_t to) {   // and into the tail, the tokens from .. to - 1
    part.store_tail(p.tail + kv_tail_at(p, s.slot, block, h, KV), x, [&](uint32_t t) {
      const uint32_t tt = block * KV_T + t;
      return tt >= from && tt < to;
    });
  };
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  fresh(blk);
  // The tail keeps the last block and the one before it. Of its two places, the first block's may still be read (the tokens
  // that it held before this call): that block's workgroup writes it, after it has read.
  const uint32_t last = end / KV_T;
  const bool kept = blk + 1 >= last && (blk == k0 || ((blk ^ k0) & 1));
  if (kept) keep(blk, s.pos, end);
  // the block's tokens before this call's: in the tail, needed where the block becomes whole
  const bool whole = (blk + 1) * KV_T <= end;
  auto before = [&](uint32_t t) { return blk * KV_T + t < s.pos; };
  if (whole && inside) part.load_tail(p.tail + kv_tail_at(p, s.slot, blk, h, KV), x, sC, before);
  // or lost, where another block has taken their place there: the codes' values are what is left of them
  const int32_t held0 = (int32_t)__builtin_amdgcn_readlane(places, 0), held1 = (int32_t)__builtin_amdgcn_readlane(places, 1);
  if (__builtin_expect(held && inside && (blk & 1 ? held1 : held0) != (int32_t)blk + 1, 0)) {
    __syncthreads();                             // (all have taken the tail's values from LDS)
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (before(part.tok(i))) x[i] = (u16x8){};
    const uint32_t page = page_of();
    if (page != 0xffffffffu) load_codes(p, part, page, h, x, sC, before);
    kv_hold(x);                                  // (a page that no call has written)
    if (kept) keep(blk, 0, s.pos);
  }
  if (whole) {
    const uint32_t page = page_of();
    const bool have = page != 0xffffffffu;
    if (inside) kv_hold(x);                      // (a tail that no call has written)
    uint32_t mx = kv_amax(x);
    for (int o = 32; o; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o, 64));
    if ((tid & 63) == 0) sMax[tid >> 6] = h_val((uint16_t)mx);
    __syncthreads();
    const float amax = fmaxf(fmaxf(sMax[0], sMax[1]), fmaxf(sMax[2], sMax[3]));
    const float sc = amax > 0.0f ? amax / 127.0f : 1.0f;
    uint8_t *codes = p.codes + kv_code_at(p, have ? page : 0u, h, KV);
    uint32_t w[8];
    kv_codes<KV>(x, sc, w);
    if constexpr (KV == 0) {
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (have) *(u32x4 *)(codes + kv_kcode(part.tok(0), part.d(2 * i))) = (u32x4){w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) *(uint32_t *)(sC + kv_lds(kv_vcode(part.tok(0), part.d(0) + j))) = w[j];
      __syncthreads();
      if (have) {
#pragma unroll
        for (int i = 0; i < 2; i++) *(u32x4 *)(codes + 16 * (tid + 256 * i)) = *(const u32x4 *)(sC + kv_lds(16 * (tid + 256 * i)));
      }
    }
    if (have && tid == 0) p.scales[kv_scale_at(p, page, h, KV)] = sc;
  }
  if (blk == k0) {
    const uint32_t cb = ((last ^ k0) & 1) ? last - 1 : last;   // the one of the last two in the first block's place
    if (last >= 1 && cb > k0 && cb * KV_T < end) {
      __syncthreads();                           // (the whole workgroup has read the first block's tokens)
      fresh(cb);
      keep(cb, s.pos, end);
    }
    if (held) {
      // What the places hold now: the last block and the one before it where this call brought tokens of theirs; no block
      // that this call wrote otherwise, and none that it left behind by going back. (Mostly as it was: nothing to write.)
      auto now = [&](uint32_t q, int32_t was) {
        const uint32_t b = ((last ^ q) & 1) ? last - 1 : last;     // the one of the last two in place q
        if ((last >= 1 || q == 0) && b >= k0 && b * KV_T < end) return (int32_t)b + 1;
        return was > (int32_t)k0 ? 0 : was;
      };
      const int32_t n0 = now(0, held0), n1 = now(1, held1);
      if (__any(n0 != held0 || n1 != held1)) {
        __syncthreads();                         // (the whole workgroup has read them)
        if (tid == 0) {
          held[0] = n0;
          held[1] = n1;
        }
      }
    }
  }
}

__global__ __launch_bounds__(256, 8) void k_kv_append(KvParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sC[2 * KV_HEAD];
  __shared__ float sMax[4];
  const uint32_t h = blockIdx.y;
  const KvItem it = kv_item<KV_T>(p, blockIdx.x);
  const KvSeq &s = it.s;
  if (!it.ok || !s.ok || s.n == 0) return;
  const uint32_t cap = p.max_pages * KV_T, k0 = s.pos / KV_T, blk = k0 + it.at;
  const uint32_t end = s.pos + s.n < cap ? s.pos + s.n : cap;
  if (blk >= p.max_pages || blk * KV_T >= end) return;
  if (blockIdx.z == 0) append_block<0>(p, s, blk, k0, end, h, sC, sMax);
  else append_block<1>(p, s, blk, k0, end, h, sC, sMax);
}

template <int KV>
__device__ void read_block(const KvParams &p, const KvSeq &s, uint32_t blk, uint32_t len, uint32_t h, uint8_t *sC) {
  const uint32_t tid = threadIdx.x, end = s.pos + s.n;
  const Part<KV> part{tid};
  u16x8 x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (u16x8){};
  if (blk < len / KV_T) {
    const uint32_t page = kv_page(p, s.slot, blk);
    if (page != 0xffffffffu) load_codes(p, part, page, h, x, sC, [](uint32_t) { return true; });
  } else if (blk == len / KV_T) {
    auto there = [&](uint32_t t) { return blk * KV_T + t < len; };
    const int32_t place = p.held && len % KV_T ? kv_held(p, s.slot, h, KV)[blk & 1] : (int32_t)blk + 1;
    part.load_tail(p.tail + kv_tail_at(p, s.slot, blk, h, KV), x, sC, there);
    if (__builtin_expect(place != (int32_t)blk + 1, 0)) {
      // a later block has taken its place, as the sequence has more tokens than the call asks for: they are in its codes
      __syncthreads();                            // (all have taken the tail's values from LDS)
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (u16x8){};
      const uint32_t page = kv_page(p, s.slot, blk);
      if (page != 0xffffffffu) load_codes(p, part, page, h, x, sC, there);
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
  __shared__ __attribute__((aligned(16))) uint8_t sC[2 * KV_HEAD];
  const uint32_t h = blockIdx.y;
  const KvItem it = kv_item<KV_T>(p, blockIdx.x);
  const KvSeq &s = it.s;
  if (!it.ok || s.n == 0) return;
  const uint32_t blk = s.pos / KV_T + it.at;
  if (blk * KV_T >= s.pos + s.n) return;
  const int32_t held = it.len;
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
