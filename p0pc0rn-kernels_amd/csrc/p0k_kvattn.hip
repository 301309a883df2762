// p0k_kvattn.hip — attention over the 8-bit key / value cache (layout: p0k_kv.h).
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j over the cached tokens j that query i sees, k = code * its block's scale
#include "p0k_device.h"
#include "p0k_kv.h"

namespace p0k {

// One wave per query row and head: a lane owns a token of a 64-token block for the scores, two d for the sums.
__global__ __launch_bounds__(64) void k_kv_attn_row(KvParams p) {
  __shared__ float sq[KV_D];
  const uint32_t r = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x, h = hq / (p.Hq / p.Hkv);
  uint32_t lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (kv_row0(p.cu, mid, p.rows) <= r) lo = mid;
    else hi = mid;
  }
  const KvSeq s = kv_seq(p, lo);
  if (r < s.r0 || r >= s.r0 + s.n) return;
  const uint32_t cap = p.max_pages * KV_T, end = s.ok ? (s.pos + s.n < cap ? s.pos + s.n : cap) : 0u, tq = s.pos + (r - s.r0);
  sq[lane] = h_val(p.K[p.krs * r + p.khs * hq + lane]);
  sq[lane + 64] = h_val(p.K[p.krs * r + p.khs * hq + lane + 64]);
  __syncthreads();
  float m = -1e30f, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (uint32_t blk = 0; blk * KV_T < end && blk * KV_T <= tq; blk++) {
    if (p.window && blk * KV_T >= p.sinks && (uint64_t)(blk + 1) * KV_T + p.window <= (uint64_t)tq + 1) continue;
    const bool open = blk == end / KV_T;
    const uint32_t page = open ? 0u : kv_page(p, s.slot, blk);
    if (page == 0xffffffffu) continue;
    const uint8_t *kc = p.codes + kv_code_at(p, page, h, 0), *vc = kc + KV_HEAD;
    const uint16_t *kt = p.tail + kv_tail_at(p, s.slot, blk, h, 0), *vt = kt + KV_HEAD;
    const float sk = open ? 1.0f : p.scales[kv_scale_at(p, page, h, 0)], sv = open ? 1.0f : p.scales[kv_scale_at(p, page, h, 1)];
    const uint32_t j = blk * KV_T + lane;
    const bool see = j < end && j <= tq && (!p.window || (uint64_t)j + p.window > tq || j < p.sinks);
    float a = 0.0f;
    for (uint32_t d = 0; d < KV_D; d++)
      a += sq[d] * (open ? (see ? h_val(kt[kv_ktail(lane, d)]) : 0.0f) : (float)(int8_t)kc[kv_kcode(lane, d)]);
    a *= sk * p.scale;
    if (p.cap > 0.0f) a = p.cap * tanhf(a / p.cap);
    a = see ? a : -1e30f;
    float mx = a;
    for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx), f = expf(m - mn), e = see ? expf(a - mn) : 0.0f;
    m = mn;
    l = l * f + e;
    o0 *= f;
    o1 *= f;
    for (uint32_t t = 0; t < KV_T; t++) {
      const float w = __shfl(e, t, 64);
      if (w == 0.0f) continue;
      o0 += w * sv * (open ? h_val(vt[kv_vtail(t, 2 * lane)]) : (float)(int8_t)vc[kv_vcode(t, 2 * lane)]);
      o1 += w * sv * (open ? h_val(vt[kv_vtail(t, 2 * lane + 1)]) : (float)(int8_t)vc[kv_vcode(t, 2 * lane + 1)]);
    }
  }
  for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o, 64);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  *(uint32_t *)(p.Ko + (uint64_t)r * p.ldo + hq * KV_D + 2 * lane) = pack2(o0 * inv, o1 * inv);
}

hipError_t launch_kv_attention(const KvParams &p, hipStream_t s) {
  if (p.rows == 0 || p.B == 0 || p.Hq == 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv_attn_row, dim3(p.rows, p.Hq), dim3(64), 0, s, p);
  return hipGetLastError();
}

}  // namespace p0k
