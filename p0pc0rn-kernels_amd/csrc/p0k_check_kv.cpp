// p0k_check_kv.cpp — host-side argument validation of the rotary positions and of the 8-bit key / value cache, and the
// translation of their argument structs into kernel parameters. Pure host code. What lies in device memory (positions, row
// offsets, slots, page numbers, lengths) cannot be checked here: the kernels hold each of it to the buffers' sizes.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/p0k.h"
#include "p0k_internal.h"
#include "p0k_kv.h"

namespace p0k {

static int fail(std::string *err, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
static int fail(std::string *err, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  if (err) *err = buf;
  return P0K_E_ARG;
}
#define NEED(cond, ...) \
  do {                  \
    if (!(cond)) return fail(err, __VA_ARGS__); \
  } while (0)
#define CHECK(call)                 \
  do {                              \
    if (int r_ = (call)) return r_; \
  } while (0)

typedef unsigned long long ull;
static constexpr uint64_t MAX_STRIDE = 1ull << 32;                  // halves; offsets into a tensor then fit 64 bits
static constexpr uint32_t MAX_ROWS = 1u << 24, MAX_SEQS = 1u << 20;  // of a call: its grids then fit the launch limits

// [off, off + need) of an operand of `size` bytes
static int fits(std::string *err, const char *op, const char *what, uint64_t off, uint64_t need, uint64_t size) {
  if (off > size || need > size - off)
    return fail(err, "%s: %s needs %llu bytes from its offset, the buffer holds %llu", op, what, (ull)need, (ull)(size > off ? size - off : 0));
  return P0K_OK;
}

// rows of H heads; out: written by the call, so no two values may share a place
static int check_heads(std::string *err, const char *op, const char *what, const void *buf, uint64_t off, uint64_t size,
                       uint64_t rs_in, uint64_t hs_in, uint32_t rows, uint32_t H, bool out, uint64_t *rs, uint64_t *hs) {
  NEED(buf != nullptr, "%s: missing %s buffer", op, what);
  *rs = rs_in ? rs_in : 128;
  NEED(off % 16 == 0 && *rs % 8 == 0 && hs_in % 8 == 0, "%s: %s: offset 16-byte aligned, strides multiples of 8", op, what);
  NEED(*rs < MAX_STRIDE && hs_in < MAX_STRIDE, "%s: %s: stride too large", op, what);
  *hs = hs_in ? hs_in : *rs * rows;
  if (rows == 0 || H == 0) return P0K_OK;
  NEED((unsigned __int128)*hs * (H - 1) < (1ull << 60), "%s: %s needs more than any buffer holds", op, what);
  if (out)
    NEED((rows == 1 || *rs >= 128) && (H == 1 || *hs >= 128) &&
             (rows == 1 || H == 1 || *rs >= *hs * (H - 1) + 128 || *hs >= *rs * (rows - 1) + 128),
         "%s: %s: rows or heads overlap (rs %llu, hs %llu)", op, what, (ull)*rs, (ull)*hs);
  return fits(err, op, what, off, (*rs * (rows - 1) + *hs * (H - 1) + 128) * 2, size);
}

// Whether two operands share no value: value d of row r and head h lies rs r + hs h + d halves behind an operand's first one.
// Operands whose ranges meet are told apart where their rows have the same stride (parts of the same rows, or of the same heads);
// where they have not, they count as overlapping.
struct RowsAt { const void *buf; uint64_t off, rs, hs; uint32_t rows, H; };
static bool apart(RowsAt a, RowsAt b) {
  typedef __int128 i128;
  if (a.rows == 0 || a.H == 0 || b.rows == 0 || b.H == 0) return true;
  if (a.rows == 1) a.rs = b.rs;
  if (b.rows == 1) b.rs = a.rs;
  if (a.H == 1) a.hs = b.hs;
  if (b.H == 1) b.hs = a.hs;
  const i128 rs = a.rs, wa = (i128)a.hs * (a.H - 1) + 128, wb = (i128)b.hs * (b.H - 1) + 128;   // from a row's first value to its last
  const i128 d = ((i128)(uintptr_t)b.buf + b.off - (i128)(uintptr_t)a.buf - a.off) / 2;          // from a's first value to b's
  if (d >= (i128)a.rs * (a.rows - 1) + wa || -d >= (i128)b.rs * (b.rows - 1) + wb) return true;
  if (a.rs != b.rs) return false;
  // a row of b is i rows on from one of a's: is there such an i with -below < at + rs i < above?
  auto meets = [&](i128 at, i128 below, i128 above) {
    const i128 lo = 1 - (i128)a.rows, hi = (i128)b.rows - 1;
    i128 i = (-below - at) / rs - 1;
    while (at + rs * i <= -below) i++;             // the first i above the lower bound
    if (i < lo) i = lo;
    return i <= hi && at + rs * i < above;
  };
  if (a.hs != b.hs) return !meets(d, wb, wa);
  for (i128 h = 1 - (i128)a.H; h < (i128)b.H; h++)
    if (meets(d + (i128)a.hs * h, 128, 128)) return false;
  return true;
}

static int check_ints(std::string *err, const char *op, const char *what, const void *buf, uint64_t off, uint64_t size, uint64_t n) {
  NEED(buf != nullptr, "%s: missing %s buffer", op, what);
  NEED(off % 4 == 0, "%s: %s offset must be a multiple of 4 bytes", op, what);
  return fits(err, op, what, off, n * 4, size);
}

static int check_batch(std::string *err, const char *op, const p0k_batch &b, KvParams *o) {
  NEED(b.rows <= MAX_ROWS && b.B <= MAX_SEQS, "%s: too many rows or sequences", op);
  CHECK(check_ints(err, op, "pos", b.pos_buf, b.pos_off, b.pos_size, b.B));
  CHECK(check_ints(err, op, "cu", b.cu_buf, b.cu_off, b.cu_size, (uint64_t)b.B + 1));
  if (b.slot_buf) CHECK(check_ints(err, op, "slot", b.slot_buf, b.slot_off, b.slot_size, b.B));
  o->pos = b.pos_buf + b.pos_off / 4;
  o->cu = b.cu_buf + b.cu_off / 4;
  o->slot = b.slot_buf ? b.slot_buf + b.slot_off / 4 : nullptr;
  o->B = b.B;
  o->rows = b.rows;
  return P0K_OK;
}

static int check_cache(std::string *err, const char *op, const p0k_kv_cache &c, uint32_t B, bool slots, KvParams *o) {
  NEED(c.Hkv > 0 && c.pages > 0 && c.slots > 0 && c.max_pages > 0, "%s: cache Hkv, pages, slots and max_pages must be positive", op);
  NEED(c.Hkv <= 65535u && c.pages <= 0x7fffffffu && c.slots <= 0x1000000u && c.max_pages <= 0x1000000u,
       "%s: cache Hkv, pages, slots or max_pages too large", op);
  NEED(slots || B <= c.slots, "%s: %u sequences on a cache of %u slots", op, B, c.slots);
  NEED(c.code_buf && c.scale_buf && c.tail_buf, "%s: missing code, scale or tail buffer", op);
  NEED(c.code_off % 16 == 0 && c.tail_off % 16 == 0 && c.scale_off % 8 == 0,
       "%s: code and tail offsets must be 16-byte aligned, the scale offset 8-byte", op);
  CHECK(fits(err, op, "code", c.code_off, p0k_kv_code_bytes(c.pages, c.Hkv), c.code_size));
  CHECK(fits(err, op, "scale", c.scale_off, p0k_kv_scale_bytes(c.pages, c.Hkv), c.scale_size));
  CHECK(fits(err, op, "tail", c.tail_off, p0k_kv_tail_bytes(c.slots, c.Hkv), c.tail_size));
  CHECK(check_ints(err, op, "table", c.table_buf, c.table_off, c.table_size, (uint64_t)c.slots * c.max_pages));
  o->codes = (uint8_t *)c.code_buf + c.code_off;
  o->scales = c.scale_buf + c.scale_off / 4;
  o->tail = (uint16_t *)((uint8_t *)c.tail_buf + c.tail_off);
  o->table = c.table_buf + c.table_off / 4;
  if (c.held_buf) {
    CHECK(check_ints(err, op, "held", c.held_buf, c.held_off, c.held_size, p0k_kv_held_bytes(c.slots, c.Hkv) / 4));
    o->held = c.held_buf + c.held_off / 4;
  }
  o->pages = c.pages; o->slots = c.slots; o->max_pages = c.max_pages; o->Hkv = c.Hkv;
  return P0K_OK;
}

#define STRUCT(op, type)                                                                                            \
  NEED(a != nullptr, op ": no arguments");                                                                          \
  NEED(a->struct_size == sizeof(type), op ": struct_size %u, this library expects %u", a->struct_size, (unsigned)sizeof(type)); \
  KvParams o = {}

int prepare_kv_append(const p0k_kv_append_args *a, KvParams *out, std::string *err) {
  STRUCT("kv_append", p0k_kv_append_args);
  CHECK(check_batch(err, "kv_append", a->batch, &o));
  CHECK(check_cache(err, "kv_append", a->cache, o.B, o.slot != nullptr, &o));
  CHECK(check_heads(err, "kv_append", "k", a->k_buf, a->k_off, a->k_size, a->k_rs, a->k_hs, o.rows, o.Hkv, false, &o.krs, &o.khs));
  CHECK(check_heads(err, "kv_append", "v", a->v_buf, a->v_off, a->v_size, a->v_rs, a->v_hs, o.rows, o.Hkv, false, &o.vrs, &o.vhs));
  o.K = (const uint16_t *)((const uint8_t *)a->k_buf + a->k_off);
  o.V = (const uint16_t *)((const uint8_t *)a->v_buf + a->v_off);
  if (out) *out = o;
  return P0K_OK;
}

int prepare_kv_read(const p0k_kv_read_args *a, KvParams *out, std::string *err) {
  STRUCT("kv_read", p0k_kv_read_args);
  CHECK(check_batch(err, "kv_read", a->batch, &o));
  CHECK(check_cache(err, "kv_read", a->cache, o.B, o.slot != nullptr, &o));
  CHECK(check_ints(err, "kv_read", "len", a->len_buf, a->len_off, a->len_size, o.B));
  CHECK(check_heads(err, "kv_read", "k", a->k_buf, a->k_off, a->k_size, a->k_rs, a->k_hs, o.rows, o.Hkv, true, &o.krs, &o.khs));
  CHECK(check_heads(err, "kv_read", "v", a->v_buf, a->v_off, a->v_size, a->v_rs, a->v_hs, o.rows, o.Hkv, true, &o.vrs, &o.vhs));
  NEED(apart({a->k_buf, a->k_off, o.krs, o.khs, o.rows, o.Hkv}, {a->v_buf, a->v_off, o.vrs, o.vhs, o.rows, o.Hkv}), "kv_read: k and v overlap");
  o.len = a->len_buf + a->len_off / 4;
  o.Ko = (uint16_t *)((uint8_t *)a->k_buf + a->k_off);
  o.Vo = (uint16_t *)((uint8_t *)a->v_buf + a->v_off);
  if (out) *out = o;
  return P0K_OK;
}

int prepare_kv_attention(const p0k_kv_attn_args *a, KvParams *out, std::string *err) {
  STRUCT("kv_attention", p0k_kv_attn_args);
  CHECK(check_batch(err, "kv_attention", a->batch, &o));
  CHECK(check_cache(err, "kv_attention", a->cache, o.B, o.slot != nullptr, &o));
  NEED(a->Hq > 0 && a->Hq <= 65535u && a->Hq % o.Hkv == 0, "kv_attention: Hq %u is not a multiple of Hkv %u (or too large)", a->Hq, o.Hkv);
  NEED(a->sinks == 0 || a->window != 0, "kv_attention: sinks without a window");
  // (a masked score is -1e30 before it is scaled, and has to stay far below the others)
  NEED(a->scale == 0.0f || (a->scale >= 0x1p-40f && a->scale <= 0x1p40f), "kv_attention: scale must be in [2^-40, 2^40] (0: 1 / sqrt(128))");
  NEED(a->cap == 0.0f || (a->cap >= 0x1p-20f && a->cap <= 0x1p20f), "kv_attention: cap must be in [2^-20, 2^20] (0: none)");
  CHECK(check_heads(err, "kv_attention", "q", a->q_buf, a->q_off, a->q_size, a->q_rs, a->q_hs, o.rows, a->Hq, false, &o.krs, &o.khs));
  NEED(a->o_buf != nullptr, "kv_attention: missing o buffer");
  o.ldo = a->ldo ? a->ldo : a->Hq * 128;
  NEED(a->o_off % 8 == 0 && o.ldo % 4 == 0 && o.ldo >= a->Hq * 128,
       "kv_attention: o offset 8-byte aligned, ldo a multiple of 4 covering Hq * 128");
  if (o.rows) CHECK(fits(err, "kv_attention", "o", a->o_off, ((uint64_t)(o.rows - 1) * o.ldo + a->Hq * 128) * 2, a->o_size));
  // (other workgroups may still read a row's queries when its results are stored)
  NEED(apart({a->q_buf, a->q_off, o.krs, o.khs, o.rows, a->Hq}, {a->o_buf, a->o_off, o.ldo, 128, o.rows, a->Hq}), "kv_attention: q and o overlap");
  o.Hq = a->Hq;
  NEED(kv_blocks_fit(o) || (kv_runs_fit(o) && !kv_long_rows(o)),
       "kv_attention: %u rows and %u sequences of %u heads over %u kv heads of max_pages %u are too many for one call", o.rows, o.B, a->Hq,
       o.Hkv, a->cache.max_pages);
  o.K = (const uint16_t *)((const uint8_t *)a->q_buf + a->q_off);
  o.Ko = (uint16_t *)((uint8_t *)a->o_buf + a->o_off);
  o.window = a->window; o.sinks = a->sinks;
  o.scale = a->scale != 0.0f ? a->scale : 0.08838834764831845f;   // 1 / sqrt(128)
  o.cap = a->cap;
  if (out) *out = o;
  return P0K_OK;
}

int prepare_rope(const p0k_rope_args *a, RopeParams *out, std::string *err) {
  NEED(a != nullptr, "rope: no arguments");
  NEED(a->struct_size == sizeof(p0k_rope_args), "rope: struct_size %u, this library expects %u", a->struct_size,
       (unsigned)sizeof(p0k_rope_args));
  RopeParams o = {};
  const p0k_batch &b = a->batch;
  NEED(b.rows <= MAX_ROWS && b.B <= MAX_SEQS, "rope: too many rows or sequences");
  NEED(a->H <= 65535u, "rope: too many heads");
  CHECK(check_ints(err, "rope", "pos", b.pos_buf, b.pos_off, b.pos_size, b.cu_buf ? b.B : b.rows));
  if (b.cu_buf) CHECK(check_ints(err, "rope", "cu", b.cu_buf, b.cu_off, b.cu_size, (uint64_t)b.B + 1));
  o.pos = b.pos_buf + b.pos_off / 4;
  o.cu = b.cu_buf ? b.cu_buf + b.cu_off / 4 : nullptr;
  o.B = b.B; o.rows = b.rows; o.H = a->H;
  CHECK(check_heads(err, "rope", "x", a->x_buf, a->x_off, a->x_size, a->x_rs, a->x_hs, b.rows, a->H, false, &o.xrs, &o.xhs));
  CHECK(check_heads(err, "rope", "y", a->y_buf, a->y_off, a->y_size, a->y_rs, a->y_hs, b.rows, a->H, true, &o.yrs, &o.yhs));
  NEED(a->x_buf != a->y_buf || a->x_off != a->y_off || (o.xrs == o.yrs && o.xhs == o.yhs), "rope: in place, x and y need the same strides");
  NEED((a->x_buf == a->y_buf && a->x_off == a->y_off) ||
           apart({a->x_buf, a->x_off, o.xrs, o.xhs, b.rows, a->H}, {a->y_buf, a->y_off, o.yrs, o.yhs, b.rows, a->H}),
       "rope: x and y overlap (in place they have the same offset and strides)");
  o.X = (const uint16_t *)((const uint8_t *)a->x_buf + a->x_off);
  o.Y = (uint16_t *)((uint8_t *)a->y_buf + a->y_off);
  o.rd = a->rd ? a->rd : 128;
  NEED(o.rd % 2 == 0 && o.rd <= 128, "rope: rd %u must be even and at most 128", a->rd);
  NEED(a->mode == P0K_ROPE_INTERLEAVED || a->mode == P0K_ROPE_HALF, "rope: mode must be 0 (interleaved) or 1 (half)");
  o.half = a->mode == P0K_ROPE_HALF;
  NEED(std::isfinite(a->mscale), "rope: mscale must be finite");
  o.mscale = a->mscale != 0.0f ? a->mscale : 1.0f;
  const double theta = a->theta != 0.0 ? a->theta : 10000.0, turn = 6.283185307179586476925286766559;
  NEED(a->freqs || (std::isfinite(theta) && theta > 0.0), "rope: theta must be positive");
  NEED(a->scaling >= P0K_ROPE_PLAIN && a->scaling <= P0K_ROPE_BANDS, "rope: scaling must be 0 (plain), 1 (linear) or 2 (bands)");
  NEED(a->scaling == P0K_ROPE_PLAIN || (std::isfinite(a->factor) && a->factor > 0.0), "rope: factor must be positive");
  NEED(a->scaling != P0K_ROPE_BANDS || (std::isfinite(a->orig) && a->orig > 0.0 && std::isfinite(a->low) && std::isfinite(a->high) && a->high > a->low),
       "rope: bands need orig > 0 and high > low");
  for (uint32_t i = 0; i < o.rd / 2; i++) {
    double f = a->freqs ? a->freqs[i] : std::pow(theta, -2.0 * i / o.rd);
    NEED(std::isfinite(f), "rope: frequency %u is not finite", i);
    if (a->scaling == P0K_ROPE_LINEAR) f /= a->factor;
    if (a->scaling == P0K_ROPE_BANDS) {
      const double u = std::fmin(1.0, std::fmax(0.0, (a->orig * f / turn - a->low) / (a->high - a->low)));
      f *= u + (1.0 - u) / a->factor;
    }
    // the fraction of a turn per token, in units of 2^-64 (a negative frequency wraps)
    double part = f / turn;
    part -= std::floor(part);
    const double hi = std::floor(std::ldexp(part, 32)), lo = std::ldexp(part, 64) - std::ldexp(hi, 32);
    o.turn[i] = ((uint64_t)hi << 32) + (uint64_t)lo;
  }
  if (out) *out = o;
  return P0K_OK;
}

}  // namespace p0k

extern "C" {
uint64_t p0k_kv_code_bytes(uint32_t pages, uint32_t Hkv) { return (uint64_t)pages * Hkv * 2 * p0k::KV_HEAD; }
uint64_t p0k_kv_scale_bytes(uint32_t pages, uint32_t Hkv) { return (uint64_t)pages * Hkv * 8; }
uint64_t p0k_kv_tail_bytes(uint32_t slots, uint32_t Hkv) { return (uint64_t)slots * Hkv * 8 * p0k::KV_HEAD; }
uint64_t p0k_kv_held_bytes(uint32_t slots, uint32_t Hkv) { return (uint64_t)slots * Hkv * 16; }
}
