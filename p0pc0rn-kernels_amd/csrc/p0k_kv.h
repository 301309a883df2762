// p0k_kv.h — the 8-bit key / value cache: its layout, the kernels' parameters and the host-side launchers.
//
// A block is 64 tokens of one sequence. A page of the pool holds a block of every kv head: for each head 8 KB of key codes
// and 8 KB of value codes, and one fp32 scale each. A code's byte is code + 128 (1 to 255): bytes 0x64 b are the f16 number
// 1024 + b, so two codes become f16 with one byte permutation and one packed subtraction. Codes lie in the order in which
// the attention kernels' matrix instructions take them, so that a wave loads its operands from memory straight into
// registers, 1 KB an instruction:
//   keys    16-byte pieces of 16 consecutive d of one token:   [half of 32 tokens][16-token tile][64 d][16 d][token % 16]
//   values  16-byte pieces of 8 tokens of d and of d + 16:     [half of 32 tokens][32 d][token group][d % 16]
// where token group q of a half holds its tokens 4 q .. 4 q + 3 and 16 + 4 q .. + 3: the eight tokens of which a lane of the
// 16x16x32 product K Q^T holds the scores (and, groups q and q + 2, those of a lane of the 32x32x16 product).
// A sequence's tail has places for two blocks (k % 2) in f16, in the same order with pieces of 8 values:
//   keys    [half][16-token tile][32 d's two steps of 8: 64 d, 8 d][16 d][token % 16]      values  [half][16 d][group][d % 16]
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "p0k_device.h"

namespace p0k {

constexpr uint32_t KV_T = 64, KV_D = 128, KV_HEAD = KV_T * KV_D;   // tokens of a block, head size, values of a block and head

struct KvParams {
  uint8_t *codes;          // [pages][Hkv][K, V][KV_HEAD]
  float *scales;           // [pages][Hkv][K, V]
  uint16_t *tail;          // [slots][2][Hkv][K, V][KV_HEAD] f16
  const int32_t *table;    // [slots][max_pages]
  int32_t *held;           // [slots][Hkv][K, V][2]: 1 + the block that the tail's place holds, 0: none (null: not kept)
  uint32_t pages, slots, max_pages, Hkv;
  const int32_t *pos, *cu, *slot, *len;   // slot, len may be null
  uint32_t B, rows;
  const uint16_t *K, *V;   // rows of K, V (append); Q in K (attention)
  uint64_t krs, khs, vrs, vhs;            // strides of K / V (attention: krs, khs of Q), in halves
  uint16_t *Ko, *Vo;       // read: rows out (same strides); attention: O in Ko
  uint32_t ldo, Hq, window, sinks;
  float scale, cap;
};

struct RopeParams {
  const uint16_t *X;
  uint16_t *Y;
  uint64_t xrs, xhs, yrs, yhs;
  const int32_t *pos, *cu;                // cu null: a position per row
  uint32_t B, rows, H, rd;
  int32_t half;
  float mscale;
  uint64_t turn[64];                      // f_i / 2 pi in units of 2^-64 turns
};

// what a sequence of the batch has in this call: rows r0 .. r0 + n - 1, its first token and its slot (ok: it has tokens)
// (down: its rows end before they begin, the batch's offsets are none)
struct KvSeq { uint32_t r0, n, pos, slot; bool ok, down; };

#ifdef __HIPCC__
__device__ __forceinline__ uint32_t kv_row0(const int32_t *cu, uint32_t b, uint32_t rows) {
  const int32_t v = cu[b];
  return v < 0 ? 0u : (uint32_t)v < rows ? (uint32_t)v : rows;
}
__device__ __forceinline__ KvSeq kv_seq(const KvParams &p, uint32_t b) {
  KvSeq s;
  s.r0 = kv_row0(p.cu, b, p.rows);
  const uint32_t r1 = kv_row0(p.cu, b + 1, p.rows);
  const int32_t pos = p.pos[b], slot = p.slot ? p.slot[b] : (int32_t)b;
  s.n = r1 > s.r0 ? r1 - s.r0 : 0u;
  s.down = r1 < s.r0;
  s.ok = pos >= 0 && slot >= 0 && (uint32_t)slot < p.slots;
  s.pos = s.ok ? (uint32_t)pos : 0u;
  s.slot = s.ok ? (uint32_t)slot : 0u;
  return s;
}
// Work items over a ragged batch: sequence b owns items f(b) .. f(b + 1) - 1 with f(b) = cu[b] / U + 2 b, at least as many as
// the blocks of U tokens that its rows touch, whatever its position; the last are idle. The sequence of an item is the
// largest b with f(b) <= item: a 64-way search of one wave down to 64 sequences, of which lane i then reads all there is to
// know about the i-th at once (one trip to memory for a batch of up to 64).
struct KvItem { KvSeq s; uint32_t at; int32_t len; bool ok; };   // at: the item's place among the sequence's
template <uint32_t U>
__device__ __forceinline__ KvItem kv_item(const KvParams &p, uint32_t item) {
  const uint32_t lane = threadIdx.x & 63u;
  auto base = [&](uint32_t b) { return kv_row0(p.cu, b, p.rows) / U + 2u * b; };
  uint32_t lo = 0, n = p.B;
  while (n > 64) {
    const uint32_t step = (n + 63u) / 64u, off = lane * step;
    const uint64_t m = __ballot(off < n && base(lo + off) <= item);
    const uint32_t k = m ? 63u - (uint32_t)__builtin_clzll(m) : 0u;
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  const uint32_t b = lo + (lane < n ? lane : n - 1u);
  const KvSeq s = kv_seq(p, b);
  const int32_t len = p.len ? p.len[b] : 0;
  const uint32_t f = s.r0 / U + 2u * b;
  const uint64_t m = __ballot(lane < n && f <= item);
  const uint32_t k = m ? 63u - (uint32_t)__builtin_clzll(m) : 0u;
  KvItem o = {};
  o.s.r0 = __builtin_amdgcn_readlane(s.r0, k);
  o.s.n = __builtin_amdgcn_readlane(s.n, k);
  o.s.pos = __builtin_amdgcn_readlane(s.pos, k);
  o.s.slot = __builtin_amdgcn_readlane(s.slot, k);
  o.s.ok = __builtin_amdgcn_readlane((uint32_t)s.ok, k) != 0;
  o.len = (int32_t)__builtin_amdgcn_readlane((uint32_t)len, k);
  const uint32_t fb = __builtin_amdgcn_readlane(f, k);
  o.ok = m != 0;
  o.at = item - fb;
  return o;
}
// byte of key / value (token t of the block, d) in a head's 8 KB of codes
__device__ __forceinline__ uint32_t kv_kcode(uint32_t t, uint32_t d) {
  return (((t >> 4) * 2 + (d >> 6)) * 4 + ((d >> 4) & 3)) * 256 + (t & 15) * 16 + (d & 15);
}
__device__ __forceinline__ uint32_t kv_vcode(uint32_t t, uint32_t d) {
  return (((t >> 5) * 4 + (d >> 5)) * 4 + ((t >> 2) & 3)) * 256 + (d & 15) * 16 + ((d >> 4) & 1) * 8 + ((t >> 4) & 1) * 4 + (t & 3);
}
// half (2-byte element) of key / value (t, d) in a head's 16 KB of the tail
__device__ __forceinline__ uint32_t kv_ktail(uint32_t t, uint32_t d) {
  return (((t >> 4) * 4 + (d >> 6) * 2 + ((d >> 3) & 1)) * 4 + ((d >> 4) & 3)) * 128 + (t & 15) * 8 + (d & 7);
}
__device__ __forceinline__ uint32_t kv_vtail(uint32_t t, uint32_t d) {
  return (((t >> 5) * 8 + (d >> 4)) * 4 + ((t >> 2) & 3)) * 128 + (d & 15) * 8 + ((t >> 4) & 1) * 4 + (t & 3);
}
__device__ __forceinline__ uint64_t kv_code_at(const KvParams &p, uint32_t page, uint32_t h, uint32_t kv) {
  return (((uint64_t)page * p.Hkv + h) * 2 + kv) * KV_HEAD;
}
__device__ __forceinline__ uint64_t kv_scale_at(const KvParams &p, uint32_t page, uint32_t h, uint32_t kv) {
  return ((uint64_t)page * p.Hkv + h) * 2 + kv;
}
__device__ __forceinline__ uint64_t kv_tail_at(const KvParams &p, uint32_t slot, uint32_t block, uint32_t h, uint32_t kv) {
  return ((((uint64_t)slot * 2 + (block & 1)) * p.Hkv + h) * 2 + kv) * KV_HEAD;
}
__device__ __forceinline__ int32_t *kv_held(const KvParams &p, uint32_t slot, uint32_t h, uint32_t kv) {
  return p.held + (((uint64_t)slot * p.Hkv + h) * 2 + kv) * 2;
}
// page of a block of a slot: 0xffffffff where there is none
__device__ __forceinline__ uint32_t kv_page(const KvParams &p, uint32_t slot, uint32_t block) {
  if (block >= p.max_pages) return 0xffffffffu;
  const int32_t v = p.table[(uint64_t)slot * p.max_pages + block];
  return v >= 0 && (uint32_t)v < p.pages ? (uint32_t)v : 0xffffffffu;
}
// the four codes of a word as f16 (exact)
__device__ __forceinline__ void kv_f16(uint32_t w, f16x2 *lo, f16x2 *hi) {
  const f16x2 k1152 = {(f16)1152.0f, (f16)1152.0f};
  *lo = as_h2(perm(0x64646464u, w, 0x04010400u)) - k1152;
  *hi = as_h2(perm(0x64646464u, w, 0x04030402u)) - k1152;
}
__device__ __forceinline__ f16x8 kv_f16x8(uint32_t a, uint32_t b) {
  f16x2 v[4];
  kv_f16(a, &v[0], &v[1]);
  kv_f16(b, &v[2], &v[3]);
  return (f16x8){v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
}
#endif

// The kernel over runs of keys counts (unit of 32 tokens, head, 16 rows) in 32 bits, by max_pages, as the lengths are not known
// here; that over blocks of rows has a workgroup of 512 threads for each block of 256 rows of a kv head, and a launch fewer than
// 2^32 threads. kv_long_rows: a sequence and kv head have more than a block on average.
inline bool kv_runs_fit(const KvParams &p) {
  return (unsigned __int128)p.max_pages * 2 * p.Hkv * ((uint64_t)p.rows * (p.Hq / p.Hkv) / 16 + p.B) < (1ull << 32);
}
inline bool kv_blocks_fit(const KvParams &p) {
  return (uint64_t)p.Hkv * ((uint64_t)p.rows * (p.Hq / p.Hkv) / 256 + p.B) < (1ull << 23);
}
inline bool kv_long_rows(const KvParams &p) { return (uint64_t)p.rows * (p.Hq / p.Hkv) > 256ull * p.B; }

// attention over runs of keys: its workspace (partial results of a workgroup's first and last group, and a counter each)
constexpr uint32_t kva_part(uint32_t rows) { return rows * (KV_D + 2); }          // floats of one partial result
uint64_t kv_attention_part_bytes(int cus);
unsigned kv_attention_counters(int cus);

hipError_t launch_rope(const RopeParams &p, hipStream_t s);
hipError_t launch_kv_append(const KvParams &p, hipStream_t s);
hipError_t launch_kv_read(const KvParams &p, hipStream_t s);
// 0: the call takes the kernel over runs of keys; else the one over blocks of rows, and the runs into which a block's keys are
// divided (more than 1 where the blocks alone do not fill the GPU); the bytes that a run leaves
unsigned kv_attention_runs(const KvParams &p, int cus);
uint64_t kv_attention_run_bytes(const KvParams &p);
// ws: part / cnt may be used; S > 1: rpart holds S runs
hipError_t launch_kv_attention(const KvParams &p, int cus, bool ws, float *part, unsigned *cnt, unsigned S, float *rpart,
                               hipStream_t s);

}  // namespace p0k
