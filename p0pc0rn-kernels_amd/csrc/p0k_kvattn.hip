// p0k_kvattn.hip — attention over the 8-bit key / value cache (layout: p0k_kv.h).
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j over the cached tokens j that query i sees, k = code * its block's scale
#include "p0k_kv.h"
#include "p0k_launch.h"

#include <algorithm>

namespace p0k {

typedef unsigned short u16;

// Two results as f16. A mean of cached values is at most 65504, but the rounding of the probabilities can carry it to where
// f16 rounds to infinity (NaN, of a query's own, stays).
__device__ __forceinline__ uint32_t pack_o(float a, float b) {
  a = fabsf(a) < 65600.0f ? fminf(fmaxf(a, -65504.0f), 65504.0f) : a;
  b = fabsf(b) < 65600.0f ? fminf(fmaxf(b, -65504.0f), 65504.0f) : b;
  return pack2(a, b);
}

// z -> tanh(z). Up to |z| = 0.75 (scores up to 3/4 of the cap: nearly all) by an odd polynomial, fitted here for the least
// largest error (1.9e-7) on that range: 6 operations at full rate, where the exponential and the reciprocal of the other form
// take a quarter of it (two chunks of 1145 queries after 12000 tokens, cap 30: 818 us with that form, 456 with this)
template <int N>
__device__ __forceinline__ void soft_cap(float (&z)[N]) {
  float mx = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) mx = fmaxf(mx, fabsf(z[i]));
  if (__any(!(mx <= 0.75f))) {
#pragma unroll
    for (int i = 0; i < N; i++) z[i] = 2.0f * sigmoid(2.0f * z[i]) - 1.0f;
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float u = z[i] * z[i];
      z[i] *= fmaf(u, fmaf(u, fmaf(u, fmaf(u, 0.012318825796f, -0.049280440068f), 0.132260913444f), -0.33323076443f), 0.999997228305f);
    }
  }
}

// What a sequence asks of the kernel: units of 32 tokens, those of the sinks [0, su) and then from unit `lo` on (0 units:
// nothing to do; a sequence that sees nothing has one that is all masked, for its rows have to be written)
struct KvWork { KvSeq s; uint32_t end, su, lo, units, blocks, io; };   // io: the first unit of the open block, by its place

template <int RB>                                 // rows of a block (a row: one query of one head)
__device__ __forceinline__ KvWork kv_work(const KvParams &p, const KvSeq &s) {
  KvWork w;
  w.s = s;
  const uint32_t cap = p.max_pages * KV_T, U32 = 32;
  w.end = w.s.ok ? (w.s.pos + w.s.n < cap ? w.s.pos + w.s.n : cap) : 0u;
  const uint32_t all = (w.end + U32 - 1) / U32;
  w.lo = 0;
  w.su = 0;
  if (p.window && w.s.pos >= p.window) {
    const uint32_t lo = (w.s.pos + 1 - p.window) / U32, su = p.sinks / U32 + (p.sinks % U32 != 0u);
    w.lo = lo < all ? lo : all;
    w.su = su < w.lo ? su : w.lo;
  }
  w.units = w.su + (all - w.lo);
  if (w.units == 0) w.units = 1;
  const uint32_t uo = w.end ? w.end / KV_T * (KV_T / U32) : 0xffffffffu;
  w.io = w.su > uo ? uo : w.lo >= uo ? w.su : uo - w.lo + w.su;
  w.blocks = (w.s.n * (p.Hq / p.Hkv) + RB - 1) / RB;
  if (w.s.n == 0) w.units = 0;
  return w;
}

// inclusive prefix sums over the wave: within rows of 16 lanes, then their sums onwards
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = dpp_add<0x111, 0xf>(v);                     // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);                     // row_bcast 15 into rows 1 and 3
  return dpp_add<0x143, 0xc>(v);                  // row_bcast 31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t rfl(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float rlf(float v, uint32_t l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l)); }

// The keys of all sequences and kv heads are one line of units of 32 tokens (sequence, head, row block, unit), of which every
// workgroup takes an equal run and every wave an equal part: a ragged batch is spread evenly, whatever its lengths. A group (sequence,
// head, row block) that lies within a wave's part is finished by that wave. One that several waves share meets in LDS: each
// leaves the part that it began with there, the wave that began the group adds them up. One that several workgroups share
// meets in the workspace: the last to arrive adds up all of them, in order, so that results do not depend on timing.
//
// A lane owns a query (of the 16 columns of a 16x16x32 product) as in S^T = K Q^T, O^T += V^T P: the scores that it holds are
// the B operand of the second product, and the cache's layout makes 16-byte loads the A operands of both. Codes are exact
// in f16; the scales stay in fp32: the keys' multiplies the scores, and O is held in units of the current block's value scale.
// P is rounded to f16 (the products have no wider operand at this rate); sums, maxima and O are fp32.
//
// HBM-bound: 48 sequences of 900 to 6000 tokens, 8 kv heads (349 MB) 64 us, of which the keys' stream takes 50 (7 TB/s); one
// sequence of 3777 tokens (7.8 MB) 9.9 us: about 2 us until the first codes are asked for, 1.4 for a unit, 6 for the exchanges.
// NB: blocks of 16 or 32 rows. 16 read the keys of 17 and more rows twice and more, but start and end sooner; the result is
// false (and nothing done) where 32 are the better choice, see k_kv_attn_split.
constexpr int KVA_NW = 8;                         // waves of a workgroup
struct KvaShared {
  __attribute__((aligned(16))) float o[KVA_NW][2 * 8 * 64 * 4];                   // parts of groups that waves share
  float m[KVA_NW][2 * 64], l[KVA_NW][2 * 64];
  uint32_t job[2][7];                                                             // groups whose last part this workgroup brought
};
template <int NB, bool CAP>
__device__ __forceinline__ bool attn_split(const KvParams &p, uint32_t ws, float *part, uint32_t *cnt, KvaShared &sh_) {
  constexpr int NW = KVA_NW;
  constexpr uint32_t RB = 16 * NB, PART = kva_part(RB);
  auto &sO = sh_.o;
  auto &sM = sh_.m, &sL = sh_.l;
  auto &sJob = sh_.job;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = rfl(tid >> 6), r16 = lane & 15, q4 = lane >> 4;
  const uint32_t rep = p.Hq / p.Hkv;
  if (tid < 2) sJob[tid][0] = 0;

  // ---- all units, and this workgroup's and wave's share of them
  // (lane i knows sequence cb + i: what it has, and the units up to its end from the chunk's start)
  KvSeq ls;
  uint32_t cb = 0, sum = 0;
  bool down = false;
  auto chunk = [&](uint32_t b0) {
    cb = b0;
    ls = KvSeq{};
    uint32_t t = 0;
    if (b0 + lane < p.B) {
      ls = kv_seq(p, b0 + lane);
      const KvWork w = kv_work<RB>(p, ls);
      t = w.units * w.blocks * p.Hkv;
    }
    down = down || __any(ls.down);
    sum = wave_scan(t);
    return __builtin_amdgcn_readlane(sum, 63);
  };
  auto work = [&](uint32_t b) {                                                   // of sequence b
    if (b - cb >= 64) chunk(b & ~63u);
    const uint32_t i = b - cb;
    KvSeq q = {};
    q.r0 = __builtin_amdgcn_readlane(ls.r0, i);
    q.n = __builtin_amdgcn_readlane(ls.n, i);
    q.pos = __builtin_amdgcn_readlane(ls.pos, i);
    q.slot = __builtin_amdgcn_readlane(ls.slot, i);
    q.ok = __builtin_amdgcn_readlane((uint32_t)ls.ok, i) != 0;
    return kv_work<RB>(p, q);
  };
  uint32_t T = chunk(0);
  for (uint32_t b0 = 64; b0 < p.B; b0 += 64) T += chunk(b0);
  if (down) T = 0;                                // offsets that decrease: sequences could share rows, and T pass 32 bits
  // the sequence of unit u < T, and its first unit
  auto find = [&](uint32_t u, uint32_t *base) {
    uint32_t at = 0, all = cb == 0 ? __builtin_amdgcn_readlane(sum, 63) : chunk(0);
    while (at + all <= u) {
      at += all;
      all = chunk(cb + 64);
    }
    const uint32_t f = (uint32_t)__builtin_ctzll(__ballot(at + sum > u));
    *base = at + (f ? __builtin_amdgcn_readlane(sum, f - 1) : 0u);
    return cb + f;
  };
  if constexpr (NB == 1) {
    // more than 64 units a workgroup, and a quarter less of them with blocks of 32 rows
    if (T > 64 * gridDim.x) {
      uint32_t T2 = 0;
      for (uint32_t b0 = 0; b0 < p.B; b0 += 64) {
        uint32_t t = 0;
        if (b0 + lane < p.B) {
          const KvWork w = kv_work<2 * RB>(p, b0 == cb ? ls : kv_seq(p, b0 + lane));
          t = w.units * w.blocks * p.Hkv;
        }
        T2 += __builtin_amdgcn_readlane(wave_scan(t), 63);
      }
      if (T2 <= T - T / 4) return false;
    }
  }
  uint32_t nwg = (T + 3) / 4;                                                     // at least 4 units each
  nwg = nwg < gridDim.x ? nwg : gridDim.x;
  // (row blocks that share their keys go to one XCD)
  const uint32_t blk = blockIdx.x, k = NB > 1 && nwg == gridDim.x && (nwg & 7u) == 0u ? (blk & 7u) * (nwg >> 3) + (blk >> 3) : blk;
  if (k >= nwg) return true;
  const uint32_t uq = T / nwg, ur = T - uq * nwg;
  auto first = [&](uint32_t i) { return uq * i + (i < ur ? i : ur); };            // the first unit of workgroup i
  auto owner = [&](uint32_t u) { return u < ur * (uq + 1) ? u / (uq + 1) : ur + (u - ur * (uq + 1)) / uq; };
  uint32_t wa = first(k), we = first(k + 1);
  if (!ws) {
    // no workspace: whole groups (a workgroup's run begins where the group of its first unit does)
    for (int i = 0; i < 2; i++) {
      uint32_t u = i ? we : wa, base;
      if (u < T) {
        const KvWork w = work(find(u, &base));
        u -= (u - base) % w.units;
      }
      (i ? we : wa) = rfl(u);
    }
    if (wa >= we) return true;
  }
  const uint32_t per = (we - wa + NW - 1) / NW;
  auto wfirst = [&](uint32_t i) { const uint32_t u = wa + i * per; return u < we ? u : we; };
  const uint32_t a = wfirst(wave), e = wfirst(wave + 1);

  f32x4 acc[NB][8];
  float m[NB], l[NB];
  auto clear = [&] {
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      m[nb] = -1.0e30f;
      l[nb] = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; d++) acc[nb][d] = (f32x4){};
    }
  };
  // this block's rows: O / l to memory
  auto put = [&](const KvWork &w, uint32_t hk, uint32_t rb) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const uint32_t row = rb * RB + nb * 16 + r16, qi = row / rep, h = hk * rep + (row - qi * rep);
      if (qi >= w.s.n) continue;
      const float inv = l[nb] > 0.0f ? 1.0f / l[nb] : 0.0f;
      u16 *o = p.Ko + (uint64_t)(w.s.r0 + qi) * p.ldo + h * KV_D + 4 * q4;
#pragma unroll
      for (int d = 0; d < 8; d++)
        *(u32x2 *)(o + 16 * d) = (u32x2){pack_o(acc[nb][d].x * inv, acc[nb][d].y * inv), pack_o(acc[nb][d].z * inv, acc[nb][d].w * inv)};
    }
  };
  const srsrc pr = stream_rsrc((const uint8_t *)part);
  // this block's rows into the workspace; the last workgroup of the group to arrive takes it on (sJob)
  auto leave = [&](const KvWork &w, uint32_t hk, uint32_t rb, uint32_t g0, uint32_t out) {
    const uint32_t base = (2 * k + out) * PART;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const uint32_t row = rb * RB + nb * 16 + r16, at = base + (nb * 16 + r16) * KV_D + 4 * q4;
      if (row / rep >= w.s.n) continue;
#pragma unroll
      for (int d = 0; d < 8; d++) sys_store128(pr, (at + 16 * d) * 4u, __builtin_bit_cast(u32x4, acc[nb][d]));
      if (q4 == 0)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, (f32x2){m[nb], l[nb]}), pr,
                                              (int)((base + RB * KV_D + 2 * (nb * 16 + r16)) * 4u), 0, SC0_SC1);
    }
    __builtin_amdgcn_s_waitcnt(0);
    const uint32_t kf = owner(g0), kl = owner(g0 + w.units - 1);
    uint32_t old = 0;
    if (lane == 0) old = __hip_atomic_fetch_add(cnt + kf, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    if (rfl(old) == kl - kf && lane == 0) {
      sJob[out][0] = 1; sJob[out][1] = kf; sJob[out][2] = kl; sJob[out][3] = hk; sJob[out][4] = rb; sJob[out][5] = w.s.r0; sJob[out][6] = w.s.n;
    }
  };

  uint32_t u = a, base = 0, b = 0, hk = 0, rb = 0, g0 = 0;
  KvWork w;
  bool tail = false;                                                              // the registers hold a group that goes on
  KvWork wi;                                                                      // wave 0: the group that an earlier workgroup began
  uint32_t hki = 0, rbi = 0, gi0 = wa;
  if (a < e) b = find(a, &base);
  while (u < e) {
    w = work(b);
    const uint32_t per_seq = w.units * w.blocks * p.Hkv;
    if (u >= base + per_seq) {                                                    // (sequences without rows have no units)
      base += per_seq;
      b++;
      continue;
    }
    const uint32_t gi = rfl((u - base) / w.units);
    hk = rfl(gi / w.blocks);
    rb = gi - hk * w.blocks;
    g0 = base + gi * w.units;
    if (g0 < wa) { wi = w; hki = hk; rbi = rb; gi0 = g0; }
    const uint32_t i0 = u - g0, i1 = (e < g0 + w.units ? e : g0 + w.units) - g0;  // units of the group, by their place in it

    // ---- the rows' queries: lane r16 holds row nb * 16 + r16, k step s = (64 d, 8 d) its d 64 (s / 2) + 16 q4 + 8 (s % 2) ..
    f16x8 qf[NB][4];
    uint32_t kmax[NB], wlo[NB];                                                   // the tokens that the row sees: below kmax, from wlo on or sinks
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      uint32_t row = rb * RB + nb * 16 + r16;
      const uint32_t last = w.s.n * rep - 1;
      row = row < last ? row : last;
      const uint32_t qi = row / rep, h = hk * rep + (row - qi * rep), t = w.s.pos + qi;
      const u16 *q = p.K + p.krs * (w.s.r0 + qi) + p.khs * h + 16 * q4;
#pragma unroll
      for (int s = 0; s < 4; s++) qf[nb][s] = *(const f16x8 *)(q + 64 * (s >> 1) + 8 * (s & 1));
      kmax[nb] = t + 1 < w.end ? t + 1 : w.end;
      wlo[nb] = p.window && t >= p.window ? t + 1 - p.window : 0u;
    }
    clear();
    float svc = 1.0f;                                                             // what O is held in units of
    const float sl2 = CAP ? p.scale / p.cap : p.scale * 1.4426950408889634f;

    auto unit_of = [&](uint32_t i) { return i < w.su ? i : i - w.su + w.lo; };
    // one unit: scores, softmax, products. kf(tt, s), vf(d): the A operands; then(): once the keys are used
    auto step = [&](uint32_t un, float sk, float sv, bool none, auto kf, auto then, auto vf) {
      const uint32_t k0 = un * 32;
      f32x4 s[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) s[nb][0] = s[nb][1] = (f32x4){};
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
#pragma unroll
        for (int st = 0; st < 4; st++) {
          const f16x8 ka = kf(tt, st);
#pragma unroll
          for (int nb = 0; nb < NB; nb++) s[nb][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qf[nb][st], s[nb][tt], 0, 0, 0);
        }
      then();
      const float f = sk * sl2;
      f16x8 pb[NB];
      const float ratio = svc / sv;
      svc = sv;
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = s[nb][i >> 2][i & 3] * f;
        if constexpr (CAP) {
          soft_cap(x);
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] *= p.cap * 1.4426950408889634f;
        }
        if (none || __any(k0 + 32 > kmax[nb] || (k0 < wlo[nb] && k0 + 32 > p.sinks))) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint32_t j = k0 + 16 * (i >> 2) + 4 * q4 + (i & 3);
            x[i] = !none && j < kmax[nb] && (j >= wlo[nb] || j < p.sinks) ? x[i] : -1.0e30f;
          }
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        // the maximum that the exponents subtract moves only when it is passed by more than 8 (P <= 256)
        const float mn = __any(mx > m[nb] + 8.0f) ? fmaxf(m[nb], mx) : m[nb];
        const float mns = mn <= -1.0e29f ? 0.0f : mn;
        float ps = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] = __builtin_amdgcn_exp2f(x[i] - mns);
          ps += x[i];
        }
        const float al = __builtin_amdgcn_exp2f(m[nb] - mn);
        l[nb] = l[nb] * al + ps;
        m[nb] = mn;
        const float g = al * ratio;
        if (__any(g != 1.0f)) {
#pragma unroll
          for (int d = 0; d < 8; d++) acc[nb][d] *= g;
        }
        pb[nb] = (f16x8){(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3], (f16)x[4], (f16)x[5], (f16)x[6], (f16)x[7]};
      }
#pragma unroll
      for (int d = 0; d < 8; d++) {
        const f16x8 va = vf(d);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) acc[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[nb], acc[nb][d], 0, 0, 0);
      }
    };

    // the open block's first unit is asked for before all others (48 sequences: 66 -> 63 us; with blocks of 32 rows there are
    // no registers to hold it)
    f16x8 ko[8], vo[8];
    const uint32_t o0 = i0 < w.io ? w.io : i0;
    auto open = [&](uint32_t i, uint32_t kv, f16x8 *to) {
      const uint32_t un = unit_of(i);
      const u16 *t = p.tail + kv_tail_at(p, w.s.slot, un >> 1, hk, kv) + (un & 1) * (KV_HEAD / 2) + lane * 8;
#pragma unroll
      for (int j = 0; j < 8; j++) to[j] = *(const f16x8 *)(t + 512 * j);
    };
    if (NB == 1 && o0 < i1) { open(o0, 0, ko); open(o0, 1, vo); }
    // (its tokens are in its codes where a later block has taken its place: the call ends before the sequence does)
    const uint32_t ob = w.end / KV_T;
    const bool codes = p.held && o0 < i1 && kv_held(p, w.s.slot, hk, 0)[ob & 1] != (int32_t)ob + 1;

    // whole blocks, up to 64 units ahead: lane i knows unit c0 + i's page and scales
    constexpr uint32_t NONE = 0xffffffffu;
    for (uint32_t c0 = i0; c0 < i1 && (c0 < w.io || codes); c0 += 64) {
      uint32_t nc = i1 - c0 < 64 ? i1 - c0 : 64;
      uint32_t pg = NONE;
      float lsk = 1.0f, lsv = 1.0f;
      if (lane < nc) {
        const uint32_t un = unit_of(c0 + lane);
        if (un * 32 < w.end) pg = kv_page(p, w.s.slot, un >> 1);
        if (pg != NONE) {
          const f32x2 sc = *(const f32x2 *)(p.scales + kv_scale_at(p, pg, hk, 0));
          lsk = sc.x;
          lsv = sc.y;
        }
      }
      if (!codes && nc > w.io - c0) nc = w.io - c0;
      // (a unit's keys are asked for when the scores of the one before it are done, its values when that one's are)
      u32x4 kc[4], vc[4];
      auto load = [&](uint32_t i, uint32_t kv, u32x4 *to) {
        const uint32_t g = __builtin_amdgcn_readlane(pg, i), un = unit_of(c0 + i);
        const uint8_t *c = p.codes + kv_code_at(p, g != NONE ? g : 0u, hk, kv) + (un & 1) * (KV_HEAD / 2) + lane * 16;
#pragma unroll
        for (int j = 0; j < 4; j++) to[j] = __builtin_nontemporal_load((const u32x4 *)(c + 1024 * j));
      };
      load(0, 0, kc);
      load(0, 1, vc);
      for (uint32_t i = 0; i < nc; i++) {
        const bool more = i + 1 < nc;
        step(unit_of(c0 + i), rlf(lsk, i), rlf(lsv, i), __builtin_amdgcn_readlane(pg, i) == NONE,
             [&](int tt, int s) { return kv_f16x8(kc[2 * tt + (s >> 1)][2 * (s & 1)], kc[2 * tt + (s >> 1)][2 * (s & 1) + 1]); },
             [&] { if (more) load(i + 1, 0, kc); },
             [&](int d) { return kv_f16x8(vc[d >> 1][2 * (d & 1)], vc[d >> 1][2 * (d & 1) + 1]); });
        if (more) load(i + 1, 1, vc);
      }
    }
    // the open block, in f16
    for (uint32_t i = codes ? i1 : o0; i < i1; i++) {
      const uint32_t un = unit_of(i);
      if (NB != 1 && i == o0) open(i, 0, ko);
      step(un, 1.0f, 1.0f, false, [&](int tt, int s) { return ko[4 * tt + s]; },
           [&] {
             if (NB != 1) open(i, 1, vo);
             if (i + 1 < i1) open(i + 1, 0, ko);
           },
           [&](int d) {
             f16x8 v = vo[d];
#pragma unroll
             for (int j = 0; j < 8; j++) v[j] = un * 32 + 16 * (j >> 2) + 4 * q4 + (j & 3) < w.end ? v[j] : (f16)0.0f;
             return v;
           });
      if (NB == 1 && i + 1 < i1) open(i + 1, 1, vo);
    }
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
      for (int d = 0; d < 8; d++) acc[nb][d] *= svc;
      l[nb] += __shfl_xor(l[nb], 16, 64);
      l[nb] += __shfl_xor(l[nb], 32, 64);
    }
    u = g0 + i1;
    if (g0 < a) {                                                                 // another wave began it
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int d = 0; d < 8; d++) *(f32x4 *)&sO[wave][((nb * 8 + d) * 64 + lane) * 4] = acc[nb][d];
        sM[wave][nb * 64 + lane] = m[nb];
        sL[wave][nb * 64 + lane] = l[nb];
      }
    } else if (g0 + w.units > e) {
      tail = true;
    } else {
      put(w, hk, rb);
    }
  }
  __syncthreads();

  // ---- groups that waves share: added to the registers, in order, from wave `from` on; true: the group ended there
  auto gather = [&](uint32_t from, uint32_t gend) {
    for (uint32_t v = from; v < (uint32_t)NW && wfirst(v) < wfirst(v + 1); v++) {
      if (wfirst(v) >= gend) return;
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        const float m2 = sM[v][nb * 64 + lane], mn = fmaxf(m[nb], m2);
        const float f1 = __builtin_amdgcn_exp2f(m[nb] - mn), f2 = __builtin_amdgcn_exp2f(m2 - mn);
        l[nb] = l[nb] * f1 + sL[v][nb * 64 + lane] * f2;
        m[nb] = mn;
#pragma unroll
        for (int d = 0; d < 8; d++) acc[nb][d] = acc[nb][d] * f1 + *(const f32x4 *)&sO[v][((nb * 8 + d) * 64 + lane) * 4] * f2;
      }
    }
  };
  if (tail) {
    gather(wave + 1, g0 + w.units);
    if (g0 + w.units <= we) put(w, hk, rb);
    else leave(w, hk, rb, g0, 1);
  }
  if (wave == 0 && gi0 < wa) {
    clear();
    gather(0, gi0 + wi.units);
    leave(wi, hki, rbi, gi0, 0);
  }
  __syncthreads();

  // ---- groups that workgroups share, whose last part came from here: threads share a row's four d over the parts
  for (int jb = 0; jb < 2; jb++) {
    if (!sJob[jb][0]) continue;
    const uint32_t kf = sJob[jb][1], kl = sJob[jb][2], hk2 = sJob[jb][3], rb2 = sJob[jb][4], np = kl - kf + 1;
    const uint32_t r0 = sJob[jb][5], left = sJob[jb][6] * rep - rb2 * RB, nrow = left < RB ? left : RB, items = nrow * 32;
    uint32_t sh = 1;                                                              // threads for each item
    while (sh < 16 && items * sh * 2 <= 64 * NW && sh * 4 <= np) sh *= 2;
    for (uint32_t it0 = 0; it0 < items; it0 += 64 * NW) {                         // (one pass where sh > 1)
      const uint32_t it = sh > 1 ? tid % items : it0 + tid, pi = sh > 1 ? tid / items : 0u;
      const bool live = pi < sh && it < items;
      const uint32_t r = it >> 5, d = (it & 31u) * 4;
      float M = -1.0e30f, L = 0.0f;
      f32x4 o = (f32x4){};
      if (live) {
        for (uint32_t s = np * pi / sh, se = np * (pi + 1) / sh; s < se; s += 8) {
          f32x4 ov[8];
          f32x2 ml[8];
#pragma unroll
          for (uint32_t x = 0; x < 8; x++) {
            const uint32_t i = s + x < se ? s + x : se - 1u, at = (2 * (kf + i) + (i == 0 ? 1u : 0u)) * PART;
            ml[x] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(pr, (int)((at + RB * KV_D + 2 * r) * 4u), 0, SC0_SC1));
            ov[x] = __builtin_bit_cast(f32x4, sys_load128(pr, (at + r * KV_D + d) * 4u));
          }
          float Mn = M;
#pragma unroll
          for (uint32_t x = 0; x < 8; x++) Mn = fmaxf(Mn, ml[x].x);
          const float f0 = __builtin_amdgcn_exp2f(M - Mn);
          o *= f0;
          L *= f0;
#pragma unroll
          for (uint32_t x = 0; x < 8; x++) {
            const float f = s + x < se ? __builtin_amdgcn_exp2f(ml[x].x - Mn) : 0.0f;
            o += f * ov[x];
            L += f * ml[x].y;
          }
          M = Mn;
        }
      }
      if (sh > 1) {
        float *so = &sO[0][0];                                                    // (the waves have taken theirs: the barrier above)
        __syncthreads();
        if (live) {
          *(f32x4 *)(so + (pi * items + it) * 4) = o;
          *(f32x2 *)(so + 64 * NW * 4 + (pi * items + it) * 2) = (f32x2){M, L};
        }
        __syncthreads();
        if (pi == 0 && live) {
          for (uint32_t q = 1; q < sh; q++) {
            const f32x2 ml = *(const f32x2 *)(so + 64 * NW * 4 + (q * items + it) * 2);
            const float Mn = fmaxf(M, ml.x), fa = __builtin_amdgcn_exp2f(M - Mn), fb = __builtin_amdgcn_exp2f(ml.x - Mn);
            o = fa * o + fb * *(const f32x4 *)(so + (q * items + it) * 4);
            L = fa * L + fb * ml.y;
            M = Mn;
          }
        }
        __syncthreads();
      }
      if (live && pi == 0) {
        const uint32_t row = rb2 * RB + r, qi = row / rep, h = hk2 * rep + (row - qi * rep);
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        *(u32x2 *)(p.Ko + (uint64_t)(r0 + qi) * p.ldo + h * KV_D + d) = (u32x2){pack_o(o.x * inv, o.y * inv), pack_o(o.z * inv, o.w * inv)};
      }
    }
    if (tid == 0) __hip_atomic_store(cnt + kf, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
  return true;
}

// Which blocks: measured over 2 head layouts, batches of 1 and 8, 1000 and 8000 keys and 8 to 256 rows, the two cross where
// blocks of 16 rows come to about 64 units a CU (24 rows, 64 heads of 8000 keys: 51.6 us against 34.8 with 32; 8 heads: 15.9
// against 22.3); up to 16 rows, 32 only add work. The lengths are known here, not on the host.
template <bool CAP>
__global__ __launch_bounds__(64 * KVA_NW, 2) void k_kv_attn_split(KvParams p, uint32_t ws, float *part, uint32_t *cnt) {
  __shared__ KvaShared sh;
  if (!attn_split<1, CAP>(p, ws, part, cnt, sh)) attn_split<2, CAP>(p, ws, part, cnt, sh);
}

// ---------------------------------------------------------------------------------------- many queries
// A workgroup owns RB = 32 NW rows of one kv head (a row: one query of one of its Hq / Hkv heads, the heads of a query side by
// side) and walks their keys, block by block: the codes come into registers two blocks ahead, become f16 on their way into
// LDS once for all of the rows, and every wave multiplies its 32 rows with them as k_attention does: S^T = K Q^T and O^T +=
// V^T P as 32x32x16 products, a lane owning a row. The cache's order of tokens is that of the score registers, so V^T needs no
// transposing read. The keys' scale multiplies the scores. The values' scale goes into the exponent: O is held in units of
// `ref`, which moves (and O with it) only when a block's scale leaves [ref, 64 ref] (P is at most 2^8 * 64 then, inside f16).
// 5003 queries of 32 heads over their own 5003 tokens: 245 us, 0.84 PFLOP/s; VALU and MFMA share the time (8 VALU per MFMA).
template <int NW, bool CAP>
__global__ __launch_bounds__(64 * NW, 2) void k_kv_attn_block(KvParams p, uint32_t items, uint32_t S, float *part) {
  constexpr uint32_t RB = 32 * NW, NP = 512 / (64 * NW);                          // pieces of 16 codes a thread moves, keys and values each
  __shared__ __attribute__((aligned(16))) f16 sK[2][KV_HEAD], sV[2][KV_HEAD];     // [8 d][token], [32 tokens][group][d]: pieces of 8
  const uint32_t tid = threadIdx.x, lane = tid & 63, gh = lane >> 5, l32 = lane & 31, wave = rfl(tid >> 6);
  const uint32_t rep = p.Hq / p.Hkv;
  // kv heads go round the XCDs, so that a head's codes stay in one L2; the longest (last) blocks first
  const uint32_t hk = blockIdx.x % p.Hkv, by = blockIdx.x / p.Hkv, item = items - 1 - by % items, run = by / items;
  auto base_of = [&](uint32_t b) { return (uint32_t)((uint64_t)kv_row0(p.cu, b, p.rows) * rep / RB) + b; };
  uint32_t b = 0;
  {
    uint32_t n = p.B;
    while (n > 1) {
      const uint32_t st = (n + 63u) / 64u, off = lane * st;
      const uint64_t m = __ballot(off < n && base_of(b + off) <= item);
      const uint32_t j = m ? 63u - (uint32_t)__builtin_clzll(m) : 0u;
      b += j * st;
      n = n - j * st < st ? n - j * st : st;
    }
    b = rfl(b);
  }
  const KvSeq s = kv_seq(p, b);
  const uint32_t ib = base_of(b), rows = s.n * rep;
  if (item < ib || (item - ib) * RB >= rows) return;
  const uint32_t row0 = (item - ib) * RB, cap = p.max_pages * KV_T;
  const uint32_t end = s.ok ? (s.pos + s.n < cap ? s.pos + s.n : cap) : 0u;
  const uint32_t rlast = row0 + RB - 1 < rows ? row0 + RB - 1 : rows - 1;
  const uint32_t ta = s.pos + row0 / rep, tb = s.pos + rlast / rep;               // the block's first and last query
  const uint32_t stop = tb + 1 < end ? tb + 1 : end, all = (stop + KV_T - 1) / KV_T;
  uint32_t lo = 0, su = 0;
  if (p.window && ta >= p.window) {
    const uint32_t l0 = (ta + 1 - p.window) / KV_T, s0 = p.sinks / KV_T + (p.sinks % KV_T != 0u);
    lo = l0 < all ? l0 : all;
    su = s0 < lo ? s0 : lo;
  }
  // tiles: [0, su), [lo, all), of which this workgroup takes its run (of four at least; fewer runs than S then)
  const uint32_t ntile = su + (all - lo), runs = S == 1 ? 1u : (ntile + 3) / 4 < S ? (ntile + 3) / 4 : S;
  const uint32_t t0 = run < runs ? (uint32_t)((uint64_t)ntile * run / runs) : 0u;
  const uint32_t nt = run < runs ? (uint32_t)((uint64_t)ntile * (run + 1) / runs) - t0 : 0u;
  auto tile_of = [&](uint32_t i) { return t0 + i < su ? t0 + i : t0 + i - su + lo; };

  uint32_t row = row0 + wave * 32 + l32;
  const bool live = row < rows;
  row = live ? row : rows - 1;
  const uint32_t qi = row / rep, h = hk * rep + (row - qi * rep), t = s.pos + qi;
  f16x8 qf[8];
  {
    const u16 *q = p.K + p.krs * (s.r0 + qi) + p.khs * h + 8 * gh;
#pragma unroll
    for (int st = 0; st < 8; st++) qf[st] = *(const f16x8 *)(q + 16 * st);
  }
  const uint32_t kmax = t + 1 < end ? t + 1 : end, wlo = p.window && t >= p.window ? t + 1 - p.window : 0u;

  // ---- moving a tile: lane i of every wave knows tile c0 + i's page and scales
  constexpr uint32_t NONE = 0xffffffffu, OPEN = 0xfffffffeu;
  uint32_t pg = NONE;
  float lsk = 1.0f, lsv = 1.0f;
  // (the open block's tokens are in its codes where a later block has taken its place: the call ends before the sequence does)
  const uint32_t ob = end / KV_T;
  const bool tail = !p.held || kv_held(p, s.slot, hk, 0)[ob & 1] == (int32_t)ob + 1;
  auto know = [&](uint32_t c0) {
    pg = NONE;
    lsk = lsv = 1.0f;
    if (c0 + lane < nt) {
      const uint32_t tl = tile_of(c0 + lane);
      pg = kv_page(p, s.slot, tl);
      if (tl == ob && tail) pg = OPEN;
      if (pg < OPEN) {
        const f32x2 sc = *(const f32x2 *)(p.scales + kv_scale_at(p, pg, hk, 0));
        lsk = sc.x;
        lsv = sc.y;
      }
    }
  };
  u32x4 ck[NP], cv[NP];
  uint32_t cg = NONE;                                                             // the page of the tile that they hold
  auto ask = [&](uint32_t i) {                                                    // codes of tile i into registers
    cg = __builtin_amdgcn_readlane(pg, i & 63);
    if (cg < OPEN) {
      const uint8_t *c = p.codes + kv_code_at(p, cg, hk, 0) + tid * 16;
#pragma unroll
      for (uint32_t j = 0; j < NP; j++) {
        ck[j] = *(const u32x4 *)(c + j * 64 * NW * 16);
        cv[j] = *(const u32x4 *)(c + KV_HEAD + j * 64 * NW * 16);
      }
    }
  };
  auto store = [&](uint32_t i, uint32_t bf) {                                     // and as f16 into LDS
    if (cg < OPEN) {
#pragma unroll
      for (uint32_t j = 0; j < NP; j++) {
        const uint32_t pc = tid + 64 * NW * j, r = pc & 15, q = (pc >> 4) & 3, k = 8 * ((pc >> 6) & 1) + 2 * q, tok = 16 * (pc >> 7) + r;
        *(f16x8 *)&sK[bf][(k * 64 + tok) * 8] = kv_f16x8(ck[j].x, ck[j].y);
        *(f16x8 *)&sK[bf][((k + 1) * 64 + tok) * 8] = kv_f16x8(ck[j].z, ck[j].w);
        const uint32_t g = 4 * (pc >> 8) + q, d = 32 * ((pc >> 6) & 3) + r;
        *(f16x8 *)&sV[bf][(g * 128 + d) * 8] = kv_f16x8(cv[j].x, cv[j].y);
        *(f16x8 *)&sV[bf][(g * 128 + d + 16) * 8] = kv_f16x8(cv[j].z, cv[j].w);
      }
    } else {
      const uint32_t tl = tile_of(i);
      const u16 *kt = p.tail + kv_tail_at(p, s.slot, tl, hk, 0);
      for (uint32_t pc = tid; pc < 1024; pc += 64 * NW) {
        const uint32_t r = pc & 15, q = (pc >> 4) & 3, st = (pc >> 6) & 3, tok = 16 * (pc >> 8) + r;
        f16x8 k = (f16x8){}, v = (f16x8){};
        const uint32_t tv = tl * KV_T + 32 * (pc >> 9) + 4 * q;                   // V: piece pc = [half][16 d][group][d % 16]
        if (cg == OPEN) {
          k = *(const f16x8 *)(kt + pc * 8);
          v = *(const f16x8 *)(kt + KV_HEAD + pc * 8);
#pragma unroll
          for (uint32_t j = 0; j < 8; j++) v[j] = tv + 16 * (j >> 2) + (j & 3) < end ? v[j] : (f16)0.0f;
        }
        *(f16x8 *)&sK[bf][((8 * (st >> 1) + 2 * q + (st & 1)) * 64 + tok) * 8] = k;
        *(f16x8 *)&sV[bf][((4 * (pc >> 9) + q) * 128 + 16 * ((pc >> 6) & 7) + r) * 8] = v;
      }
    }
  };

  f32x16 oacc[4];
#pragma unroll
  for (int i = 0; i < 4; i++) oacc[i] = (f32x16){};
  float m = -1.0e30f, l = 0.0f, ref = 0.0f;                                       // ref 0: none yet
  const float sl2 = CAP ? p.scale / p.cap : p.scale * 1.4426950408889634f;
  uint32_t gc = NONE;
  float sk = 1.0f, sv = 1.0f, skn = 1.0f, svn = 1.0f;
  if (nt) {
    know(0);
    ask(0);
    store(0, 0);
    gc = cg;
    sk = rlf(lsk, 0);
    sv = rlf(lsv, 0);
    if (nt > 1) ask(1);
  }
  for (uint32_t i = 0; i < nt; i++) {
    const uint32_t bf = i & 1;
    __syncthreads();                                                              // tile i is there, tile i - 1 is done with
    const uint32_t gi = gc;
    if (i + 1 < nt) {
      store(i + 1, bf ^ 1);
      gc = cg;
      skn = rlf(lsk, (i + 1) & 63);
      svn = rlf(lsv, (i + 1) & 63);
      if (i + 2 < nt) {
        if (((i + 2) & 63) == 0) know(i + 2);
        ask(i + 2);
      }
    }
    f32x16 sacc[2];
    sacc[0] = (f32x16){};
    sacc[1] = (f32x16){};
#pragma unroll
    for (int st = 0; st < 8; st++)
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        const f16x8 a = *(const f16x8 *)&sK[bf][((2 * st + gh) * 64 + 32 * kb + l32) * 8];
        sacc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[st], sacc[kb], 0, 0, 0);
      }
    const float f = sk * sl2;
    const uint32_t k0 = tile_of(i) * KV_T;
    float sf = f;
    if constexpr (CAP) {
      float z[32];
#pragma unroll
      for (int r = 0; r < 32; r++) z[r] = sacc[r >> 4][r & 15] * f;
      soft_cap(z);
#pragma unroll
      for (int r = 0; r < 32; r++) sacc[r >> 4][r & 15] = z[r];
      sf = p.cap * 1.4426950408889634f;
    }
    if (gi == NONE || __any(k0 + KV_T > kmax || (k0 < wlo && k0 + KV_T > p.sinks))) {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const uint32_t j = k0 + 32 * kb + 8 * (r >> 2) + 4 * gh + (r & 3);
          sacc[kb][r] = gi != NONE && j < kmax && (j >= wlo || j < p.sinks) ? sacc[kb][r] : -1.0e30f;
        }
    }
    float mx = -1.0e30f;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++) mx = fmaxf(mx, sacc[kb][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mxl = mx <= -1.0e29f ? -1.0e30f : mx * sf;
    const float mn = __any(mxl > m + 8.0f) ? fmaxf(m, mxl) : m;
    float scale_o = 1.0f;
    if (sv < ref || sv > 64.0f * ref) {                                           // (uniform)
      const float nr = 0.125f * sv;
      scale_o = ref / nr;
      ref = nr;
    }
    const float lr = __builtin_amdgcn_logf(sv / ref);                             // log2; 0 .. 6
    const float mns = (mn <= -1.0e29f ? 0.0f : mn) - lr;
    float ps = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float e = __builtin_amdgcn_exp2f(fmaf(sacc[kb][r], sf, -mns));
        sacc[kb][r] = e;
        ps += e;
      }
    if (scale_o != 1.0f || __any(mn != m)) {
      const float al = __builtin_amdgcn_exp2f(m - mn);
      l *= al;
      const float g = al * scale_o;
#pragma unroll
      for (int db = 0; db < 4; db++) oacc[db] *= g;
    }
    m = mn;
    l = fmaf(ps, __builtin_amdgcn_exp2f(-lr), l);
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const f16x8 bp = {(f16)sacc[kb][4 * c + 0], (f16)sacc[kb][4 * c + 1], (f16)sacc[kb][4 * c + 2], (f16)sacc[kb][4 * c + 3],
                          (f16)sacc[kb][4 * c + 8], (f16)sacc[kb][4 * c + 9], (f16)sacc[kb][4 * c + 10], (f16)sacc[kb][4 * c + 11]};
#pragma unroll
        for (int db = 0; db < 4; db++) {
          const f16x8 av = *(const f16x8 *)&sV[bf][((4 * kb + 2 * c + gh) * 128 + 32 * db + l32) * 8];
          oacc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, bp, oacc[db], 0, 0, 0);
        }
      }
    sk = skn;
    sv = svn;
  }

  const float lt = l + __shfl_xor(l, 32, 64);
  if (!live) return;
  if (S > 1) {
    // one of several runs: its part by (run, row, head), and what it is: the maximum and sum of the row; sum -1: not there.
    // Where there is only one run after all, its rows are finished here (-2)
    float *pr = part + ((uint64_t)run * p.rows * p.Hq + (uint64_t)(s.r0 + qi) * p.Hq + h) * (KV_D + 2);
    if (gh == 0) *(f32x2 *)pr = (f32x2){m, run >= runs ? -1.0f : runs <= 1 ? -2.0f : lt};
    if (run >= runs && run) return;
    if (runs > 1) {
#pragma unroll
      for (int db = 0; db < 4; db++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          float *o = pr + 2 + 32 * db + 8 * g4 + 4 * gh;
          *(f32x2 *)o = (f32x2){oacc[db][4 * g4] * ref, oacc[db][4 * g4 + 1] * ref};
          *(f32x2 *)(o + 2) = (f32x2){oacc[db][4 * g4 + 2] * ref, oacc[db][4 * g4 + 3] * ref};
        }
      return;
    }
  }
  const float inv = lt > 0.0f ? ref / lt : 0.0f;
  u16 *o = p.Ko + (uint64_t)(s.r0 + qi) * p.ldo + h * KV_D + 4 * gh;
#pragma unroll
  for (int db = 0; db < 4; db++)
#pragma unroll
    for (int g4 = 0; g4 < 4; g4++)
      *(u32x2 *)(o + 32 * db + 8 * g4) = (u32x2){pack_o(oacc[db][4 * g4] * inv, oacc[db][4 * g4 + 1] * inv),
                                                pack_o(oacc[db][4 * g4 + 2] * inv, oacc[db][4 * g4 + 3] * inv)};
}

// The runs of k_kv_attn_block together: a half wave for a row of a head, four d a thread. With offsets that decrease not every
// row has parts, and two sequences may have left theirs in the same place: nothing to join then. (B is small here: the blocks of
// all sequences and heads are fewer than two a CU.)
__global__ __launch_bounds__(256) void k_kv_attn_join(KvParams p, uint32_t S, const float *part) {
  bool down = false;
  for (uint32_t b = threadIdx.x; b < p.B; b += 256) down |= kv_row0(p.cu, b + 1, p.rows) < kv_row0(p.cu, b, p.rows);
  if (__syncthreads_or(down)) return;
  const uint64_t it = (uint64_t)blockIdx.x * 256 + threadIdx.x, rh = it >> 5, n = (uint64_t)p.rows * p.Hq;
  if (rh >= n) return;
  const uint32_t r = (uint32_t)(rh / p.Hq), h = (uint32_t)(rh - (uint64_t)r * p.Hq), d = 4 * ((uint32_t)it & 31u);
  if (r < kv_row0(p.cu, 0, p.rows) || r >= kv_row0(p.cu, p.B, p.rows)) return;
  const float *pr = part + rh * (KV_D + 2);
  const uint64_t step = n * (KV_D + 2);
  float M = -1.0e30f, L = 0.0f;
  f32x4 o = (f32x4){};
  for (uint32_t i = 0; i < S; i++, pr += step) {
    const f32x2 ml = *(const f32x2 *)pr;
    if (ml.y == -2.0f) return;
    if (ml.y == -1.0f) break;
    const f32x2 a = *(const f32x2 *)(pr + 2 + d), b = *(const f32x2 *)(pr + 4 + d);
    const float mn = fmaxf(M, ml.x), f1 = __builtin_amdgcn_exp2f(M - mn), f2 = __builtin_amdgcn_exp2f(ml.x - mn);
    o = o * f1 + (f32x4){a.x, a.y, b.x, b.y} * f2;
    L = L * f1 + ml.y * f2;
    M = mn;
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  *(u32x2 *)(p.Ko + (uint64_t)r * p.ldo + h * KV_D + d) = (u32x2){pack_o(o.x * inv, o.y * inv), pack_o(o.z * inv, o.w * inv)};
}

uint64_t kv_attention_part_bytes(int cus) {
  return (uint64_t)cus * 2 * kva_part(32) * sizeof(float);
}
unsigned kv_attention_counters(int cus) { return (unsigned)cus; }

// Which kernel: blocks of 256 rows where a sequence and kv head have more than that on average and all rows of all heads are
// more than 20 a CU; runs of keys otherwise. Measured over 2 head layouts, batches of 1 and 8, 1000 and 8000 keys, 16 to 1024
// rows: 8 heads x 512 rows, 8000 keys: runs 46.5 us, blocks 50.6; x 768: 60.2 and 52.7; 64 heads x 256 rows: 140 and 142 (1000
// keys: 25.7 and 45.6); x 384: 210 and 157 (37 and 51). And where the runs would be too many to count.
static bool by_blocks(const KvParams &p, int cus) {
  return (kv_long_rows(p) && (uint64_t)p.rows * p.Hq > 20ull * cus) || !kv_runs_fit(p);
}
constexpr uint32_t KVA_BLOCK = 256;               // rows of a block of k_kv_attn_block
static uint32_t block_items(const KvParams &p) { return (uint32_t)((uint64_t)p.rows * (p.Hq / p.Hkv) / KVA_BLOCK + p.B); }

// Runs of a block's keys: two workgroups for each CU between all blocks, eight at most (two chunks of 1145 queries after 12000
// keys, 152 blocks: one run 456 us, two 349, three 327, four 315)
unsigned kv_attention_runs(const KvParams &p, int cus) {
  if (!by_blocks(p, cus)) return 0;
  if (p.max_pages < 8) return 1;
  const uint64_t groups = (uint64_t)block_items(p) * p.Hkv;
  return groups >= 2u * cus ? 1u : std::min(8u, (unsigned)((2u * cus + groups - 1) / groups));
}
uint64_t kv_attention_run_bytes(const KvParams &p) { return (uint64_t)p.rows * p.Hq * (KV_D + 2) * sizeof(float); }

hipError_t launch_kv_attention(const KvParams &p, int cus, bool ws, float *part, unsigned *cnt, unsigned S, float *rpart, hipStream_t s) {
  if (p.rows == 0 || p.B == 0 || p.Hq == 0) return hipSuccess;
  if (S) {
    const uint32_t items = block_items(p);
    const dim3 grid(items * p.Hkv * S), block(512);
    if (p.cap > 0.0f) hipLaunchKernelGGL((k_kv_attn_block<8, true>), grid, block, 0, s, p, items, S, rpart);
    else hipLaunchKernelGGL((k_kv_attn_block<8, false>), grid, block, 0, s, p, items, S, rpart);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || S == 1) return e;
    const uint64_t threads = (uint64_t)p.rows * p.Hq * 32;
    hipLaunchKernelGGL(k_kv_attn_join, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, s, p, S, rpart);
    return hipGetLastError();
  }
  const dim3 grid(cus), block(64 * KVA_NW);
  if (p.cap > 0.0f) hipLaunchKernelGGL(k_kv_attn_split<true>, grid, block, 0, s, p, ws ? 1u : 0u, part, cnt);
  else hipLaunchKernelGGL(k_kv_attn_split<false>, grid, block, 0, s, p, ws ? 1u : 0u, part, cnt);
  return hipGetLastError();
}

}  // namespace p0k
