// Host side of the paged 8-bit KV cache's operators (megakernel_op_qk_norm_rope,
// megakernel_op_kv8_*): argument checks and launches.  Every call only
// enqueues on the caller's stream: no allocation, no copy, no wait, so it can
// be captured into a graph.  Lengths and block tables stay on the device; the
// grids come from the row count alone, and each workgroup finds its sequence
// there.
#include "mk_kv8.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "megakernel.h"
#include "mk_host.h"

namespace mk {
namespace kv8 {

static bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

static int type_size(int type) { return type == MK_TYPE_F32 ? 4 : type == MK_TYPE_BF16 ? 2 : 0; }

// A tensor of rows: type, alignment for 16-byte accesses, and strides that
// keep the heads of one token apart.
static bool rows_ok(const char* op, const char* name, const megakernel_rows* r, int heads, int head_dim, bool bf16_only) {
  if (!r || !r->p) {
    set_err("%s: null %s", op, name);
    return false;
  }
  const int sz = type_size(r->type);
  if (!sz || (bf16_only && r->type != MK_TYPE_BF16)) {
    set_err("%s: %s has type %d (%s)", op, name, r->type, bf16_only ? "bf16 only" : "bf16 or fp32");
    return false;
  }
  if (!aligned(r->p, 16) || r->token_stride * sz % 16 || r->head_stride * sz % 16) {
    set_err("%s: %s needs 16-byte aligned rows (strides %lld, %lld)", op, name, r->token_stride, r->head_stride);
    return false;
  }
  if (r->token_stride < 0 || r->head_stride < 0 || (heads > 1 && r->head_stride < head_dim)) {
    set_err("%s: %s strides %lld, %lld overlap rows of %d", op, name, r->token_stride, r->head_stride, head_dim);
    return false;
  }
  return true;
}

// Rows that are written must not lie on each other.
static bool apart(const char* op, const char* name, const megakernel_rows* r, int heads, int head_dim, long long tokens) {
  const long long t = r->token_stride, h = r->head_stride;
  const bool token_major = t >= (heads - 1) * h + head_dim, head_major = heads > 1 && h >= (tokens - 1) * t + head_dim && t >= head_dim;
  if (tokens > 1 && !token_major && !head_major) {
    set_err("%s: rows of %s overlap (strides %lld, %lld)", op, name, t, h);
    return false;
  }
  return true;
}

// Two tensors, one of them written, that cannot be the same.
static bool two(const char* op, const char* names, const megakernel_rows* a, const megakernel_rows* b) {
  if (a->p != b->p) return true;
  set_err("%s: %s must not be the same rows", op, names);
  return false;
}

static bool cache_ok(const char* op, const megakernel_kv8_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
    set_err("%s: null cache pointer", op);
    return false;
  }
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) {
    set_err("%s: cache codes need 16-byte alignment, scales 4", op);
    return false;
  }
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) {
    set_err("%s: block=%d (16, 32, 64 or 128 positions)", op, c->block);
    return false;
  }
  if (c->head_dim != 64 && c->head_dim != 128) {
    set_err("%s: head_dim=%d (64 or 128)", op, c->head_dim);
    return false;
  }
  if (c->n_blocks < 1 || c->n_kv < 1 || c->n_kv > 1024) {
    set_err("%s: n_blocks=%d (at least 1), n_kv=%d (1..1024)", op, c->n_blocks, c->n_kv);
    return false;
  }
  return true;
}

static bool batch_ok(const char* op, const megakernel_kv8_batch* b, int block) {
  if (!b || !b->table || !b->q_start || !b->kv_len) {
    set_err("%s: null batch pointer", op);
    return false;
  }
  if (!aligned(b->table, 4) || !aligned(b->q_start, 4) || !aligned(b->kv_len, 4)) {
    set_err("%s: batch arrays need 4-byte alignment", op);
    return false;
  }
  if (b->n_seq < 0 || b->n_seq > (1 << 20) || b->n_tokens < 0 || b->n_tokens > (1 << 27) || b->max_kv < 0) {
    set_err("%s: n_seq=%d (0..2^20), n_tokens=%d (0..2^27), max_kv=%d (>= 0)", op, b->n_seq, b->n_tokens, b->max_kv);
    return false;
  }
  if (b->table_width < 1 || (long long)b->table_width * block > (1ll << 30)) {
    set_err("%s: table_width=%d blocks of %d positions (at least 1 block, at most 2^30 positions)", op, b->table_width, block);
    return false;
  }
  return true;
}

static Cache cache_of(const megakernel_kv8_cache* c) {
  Cache r;
  r.k = static_cast<uint8_t*>(c->k);
  r.v = static_cast<uint8_t*>(c->v);
  r.ks = c->k_scale;
  r.vs = c->v_scale;
  r.n_blocks = c->n_blocks;
  r.n_kv = c->n_kv;
  r.lb = __builtin_ctz((unsigned)c->block);
  return r;
}
static Batch batch_of(const megakernel_kv8_batch* b) {
  return Batch{b->table, b->q_start, b->kv_len, b->n_seq, b->table_width, b->n_tokens};
}
static Rows rows_of(const megakernel_rows* r) { return Rows{r->p, r->token_stride, r->head_stride}; }

// HIP bounds a grid to 2^32 - 1 threads.
static bool grid_ok(const char* op, long long groups) {
  if (groups * 256 > 0xffffffffll) {
    set_err("%s: too many rows for one launch (%lld workgroups)", op, groups);
    return false;
  }
  return true;
}

template <class T>
struct Same {
  typedef T type;
};
// What a kernel's launch returns; no error that an earlier call left is taken
// for its own.
template <class... P>
static hipError_t launch(void (*kern)(P...), long long groups, int threads, hipStream_t st, typename Same<P>::type... args) {
  void* a[] = {&args...};
  return hipLaunchKernel(reinterpret_cast<const void*>(kern), dim3((unsigned)groups), dim3(threads), a, 0, st);
}

static int launched(const char* op, hipError_t e) {
  if (e == hipSuccess) return 0;
  (void)hipGetLastError();  // reported here
  set_err("%s: launch failed: %s", op, hipGetErrorString(e));
  return -1;
}

// Most workgroup items that the blocks of n_tokens rows make.
static long long block_items(const megakernel_kv8_batch* b, int block) {
  const long long n = b->n_tokens, m = n / block + 2ll * b->n_seq;
  return n < m ? n : m;
}
// Most tiles of `rows` query rows.
static long long most_row_tiles(const megakernel_kv8_batch* b, int group, int rows) {
  const long long n = b->n_tokens, m = n * group / rows + b->n_seq, each = n * ((group + rows - 1) / rows);
  return each < m ? each : m;
}

// How the attention of a batch is launched.
struct Plan {
  bool use[2];                   // attn_rows, attn_tile
  int few;                       // as in Attn
  int waves;                     // of attn_rows's workgroups
  int lr[2], target[2], least[2];
  long long items[2], slots[2];  // most items, and partials, per KV head
};

// Lengths are on the device, so what is chosen here goes by the sizes that
// the host has: rows, sequences, and how long contexts may get (max_kv).
// Every choice is right for any lengths.
static Plan plan(const megakernel_kv8_cache* c, const megakernel_kv8_batch* b, int n_q) {
  Plan p{};
  const int group = n_q / c->n_kv;
  const bool d64 = c->head_dim == 64;
  const long long rows = (long long)b->n_tokens * group;
  const long long kv = b->max_kv ? b->max_kv : (long long)b->table_width * c->block, steps = (kv + TILE - 1) / TILE;
  // Which kernel takes a batch.  attn_rows reads a context once for every 16
  // rows but starts fast; attn_tile has two to three times the rate once its
  // 128-row tiles fill the chip, and before that waits for its longest tile, or
  // for the join of splits.  They are even at nearly as many rows as give every
  // CU a tile (head_dim 128: two CUs of three), or at fewer that work longer.
  // us of attn_rows / attn_tile, 8 KV heads: head_dim 64, 4,096 rows without a
  // past in one sequence 37 / 41, in four 18 / 16, in 16 11 / 10, with 1,000
  // positions before them in four 37 / 35; 2,048 rows after 4,000 53 / 57,
  // 1,024 after 8,000 47 / 51, 512 after 16,000 44 / 51, 1,024 76 / 71; 128:
  // 2,048 rows in one sequence 23 / 33, in two 16 / 21, in four 13 / 15, 4,096
  // 58 / 57, 34 / 34, 29 / 23; 1,024 after 4,000 53 / 50, 2,048 103 / 75, 256
  // after 8,000 38 / 35.
  const long long cap = d64 ? 3584 : 2560, work = (d64 ? 7ll << 15 : 1ll << 16) / steps;
  const long long even = (work < cap ? work : cap) * 8 / c->n_kv;
  if (rows <= even || rows <= 16ll * b->n_seq) {
    p.use[FEW] = true;
    p.few = 0x7fffffff;
  } else {
    // In a batch that fills the chip a tile costs as much as 64 rows of
    // attn_rows, or 32 (64 sequences, us of attn_rows / attn_tile; head_dim 64
    // after 1,000 positions 62 rows each 29 / 34, after 200 17 / 15, without a
    // past 14 / 9, 34 rows 23 / 31, 13 / 14, 11 / 8; 128: 62 rows 63 / 52, 31 /
    // 22, 24 / 15, 34 rows 49 / 49, 24 / 20, 18 / 13, 32 rows 39 / 49, 18 / 20,
    // 13 / 12).
    p.use[MANY] = true;
    p.few = b->n_seq == 1 ? 0 : d64 && steps > 8 ? 64 : 32;
    p.use[FEW] = group <= p.few;  // one token has `group` rows
  }
  p.lr[FEW] = 4, p.lr[MANY] = 7;
  p.least[FEW] = 8, p.least[MANY] = 4;
  if (p.use[FEW]) {
    long long tiles = most_row_tiles(b, group, ROWS);
    const long long most = (long long)b->n_seq * ((p.few + ROWS - 1ll) / ROWS);
    if (tiles > most) tiles = most;
    // Splitting costs a second kernel and a second start (5 us), and saves
    // steps on a CU that has neighbours idle: worth it from about 40 steps of
    // 8 KB or 16 of 16 KB on one sequence, later the more CUs are busy anyway
    // (us unsplit / split; head_dim 64: one sequence of 1,024 positions 6.3 /
    // 9.3, of 4,096 12.0 / 9.3, four of 2,048 8.3 / 9.5, 16 of 4,096 15.2 /
    // 18.9; 128: 1,024 9.6 / 10.7, 4,096 23.3 / 10.8, four of 2,048 15.6 /
    // 12.3, 16 of 4,096 37.4 / 32.6).  Split work goes to workgroups of four
    // waves, two for every CU.  Sequences end inside a part, which makes half a
    // part more for every row tile: with these over the two, some CUs would
    // start a third when the others end (16 of 700 to 8,191, 128: 37.6, now
    // 35.0; 12 of 500 to 20,000: 58 / 54; four of 8,000 alike 19.3 / 19.9).
    // `tiles` is a bound from sizes alone: beside a prompt it counts every
    // sequence as if it had `few` rows, so with 8 KV heads nothing is split
    // from 8 sequences of head_dim 64 on, or 16 of 128, and of single tokens
    // alone from about 30.  One context of 32,768 among others of 512 is then
    // walked whole: 31 single tokens 70 us (head_dim 128 190), 16, split, 15
    // (22); beside a prompt of 1,024 tokens 8 of head_dim 64 113, 6, split, 34,
    // and 15 of 128 274, 14, split, 53.
    const long long units = tiles * c->n_kv;
    if (units < 256 && steps * (256 - units) > 256 * (d64 ? 40 : 16)) {
      p.target[FEW] = (512 + c->n_kv - 1) / c->n_kv - (b->n_seq > 1 ? (int)tiles / 2 : 0);
      p.waves = 4;
    } else {
      // Whole contexts: as many waves as the steps occupy, fewer where
      // workgroups are many (us with 8 / 4 / 2 waves, head_dim 64; 256
      // workgroups of 16 steps 8.0 / 8.9 / 12.7, of 64 16 / 20 / 34; 512 of 24
      // 14.2 / 12.8 / 18.9, of 64 27 / 29 / 46; 1,024 of 4 14 / 10 / 8.5, of 16
      // 19 / 13 / 15, of 64 53 / 50 / 52; 4,096 of 1 50 / 25 / 18).
      const long long low = (rows / ROWS > b->n_seq ? rows / ROWS : b->n_seq) * c->n_kv;
      p.waves = low >= 1024 ? (steps <= 8 ? 2 : 4) : steps <= (low > 256 ? 48 : 8) ? 4 : 8;
    }
    p.items[FEW] = tiles + p.target[FEW];
    p.slots[FEW] = 2ll * p.target[FEW];
  }
  if (p.use[MANY]) {
    long long tiles = most_row_tiles(b, group, TILE_ROWS);
    const long long most = rows / TILE_ROWS + rows / (p.few + 1);  // of sequences with more rows than `few`
    if (tiles > most) tiles = most;
    // Three workgroups of head_dim 64 fit a CU, two of 128 (1,024 tokens at the
    // end of 8,192 and 32,768 positions, us in 512 / 768 parts: 64 74, 217 /
    // 68, 202; 128 100, 316 / 109, 326).  Where the row tiles do not fill them,
    // contexts are split if they are long: the partials' way through memory and
    // the join cost 10 us, more for more rows (us unsplit / split, one sequence,
    // head_dim 64: 1,024 tokens 23 / 32, after 1,000 positions 40 / 39, after
    // 4,000 89 / 57; 2,048 tokens 41 / 54, 59 / 65, 109 / 102; 128: 31 / 37,
    // 56 / 46, 122 / 75; 56 / 64, 82 / 80, 148 / 135).
    const long long units = rows / TILE_ROWS * c->n_kv;
    if (steps * (512 - units) > 5120 + 32 * units) p.target[MANY] = ((d64 ? 768 : 512) + c->n_kv - 1) / c->n_kv;
    p.items[MANY] = tiles + p.target[MANY];
    p.slots[MANY] = 2ll * p.target[MANY];
  }
  return p;
}

static long long part_floats(const Plan& p, int k, int n_kv, int head_dim) { return p.slots[k] * n_kv * head_dim << p.lr[k]; }
static long long part_bytes(const Plan& p, int k, int n_kv, int head_dim) {
  return part_floats(p, k, n_kv, head_dim) * 4 + (p.slots[k] * n_kv << p.lr[k]) * 8;
}
static long long workspace(const Plan& p, int n_kv, int head_dim) {
  return part_bytes(p, FEW, n_kv, head_dim) + part_bytes(p, MANY, n_kv, head_dim);
}

static bool heads_ok(const char* op, int n_q, int n_kv) {
  if (n_kv < 1 || n_kv > 1024 || n_q < 1 || n_q > 1024 || n_q % n_kv) {
    set_err("%s: n_q=%d must be a multiple of n_kv=%d (both 1..1024)", op, n_q, n_kv);
    return false;
  }
  return true;
}

// Pieces of 4 rows x 8 dimensions of one block and head.
static int block_pieces(const megakernel_kv8_cache* c) { return c->block / 4 * (c->head_dim / 8); }

template <int D>
static hipError_t launch_append(int pieces, bool f32, long long groups, hipStream_t st, Cache c, Batch b, Rows k, Rows v) {
  auto go = [&](auto kern) { return launch(kern, groups, 256, st, c, b, k, v); };
  if constexpr (D == 64)
    if (pieces == 32) return f32 ? go(append<D, 32, 1, true>) : go(append<D, 32, 1, false>);
  if (pieces == 64) return f32 ? go(append<D, 64, 1, true>) : go(append<D, 64, 1, false>);
  if (pieces == 128) return f32 ? go(append<D, 128, 1, true>) : go(append<D, 128, 1, false>);
  if constexpr (D == 128)
    if (pieces == 512) return f32 ? go(append<D, 256, 2, true>) : go(append<D, 256, 2, false>);
  return f32 ? go(append<D, 256, 1, true>) : go(append<D, 256, 1, false>);
}

}  // namespace kv8
}  // namespace mk

using namespace mk;
using namespace mk::kv8;

extern "C" {

int megakernel_op_qk_norm_rope(const megakernel_rows* q, const megakernel_rows* k, const void* q_gain,
                               const void* k_gain, const float* inv_freq, const int* pos, const megakernel_rows* q_out,
                               const megakernel_rows* k_out, int n_tokens, int n_q, int n_kv, int head_dim, float eps,
                               void* stream) {
  const char* op = "op_qk_norm_rope";
  if (head_dim != 64 && head_dim != 128) {
    set_err("%s: head_dim=%d (64 or 128)", op, head_dim);
    return -1;
  }
  if (n_q < 1 || n_q > 1024 || n_kv < 1 || n_kv > 1024 || n_tokens < 0 || n_tokens > (1 << 27)) {
    set_err("%s: n_q=%d, n_kv=%d (both 1..1024), n_tokens=%d (0..2^27)", op, n_q, n_kv, n_tokens);
    return -1;
  }
  if (!(eps >= 0.f)) {
    set_err("%s: eps=%g must be at least 0", op, eps);
    return -1;
  }
  if (!rows_ok(op, "q", q, n_q, head_dim, false) || !rows_ok(op, "k", k, n_kv, head_dim, false) ||
      !rows_ok(op, "q_out", q_out, n_q, head_dim, false) || !rows_ok(op, "k_out", k_out, n_kv, head_dim, false) ||
      !apart(op, "q_out", q_out, n_q, head_dim, n_tokens) || !apart(op, "k_out", k_out, n_kv, head_dim, n_tokens))
    return -1;
  if (!q_gain || !k_gain || !inv_freq || !pos || !aligned(q_gain, 16) || !aligned(k_gain, 16) || !aligned(inv_freq, 4) ||
      !aligned(pos, 4)) {
    set_err("%s: null or unaligned gains (16 bytes), inv_freq or pos (4)", op);
    return -1;
  }
  if (q->type != k->type || q_out->type != k_out->type) {
    set_err("%s: q and k must have one type (%d, %d), and so must q_out and k_out (%d, %d)", op, q->type, k->type,
            q_out->type, k_out->type);
    return -1;
  }
  // in place: a lane writes what it alone has read, if the layout is the same
  auto moved = [](const megakernel_rows* a, const megakernel_rows* b) {
    return a->p == b->p && (a->type != b->type || a->token_stride != b->token_stride || a->head_stride != b->head_stride);
  };
  if (moved(q, q_out) || moved(k, k_out)) {
    set_err("%s: an output in place of its input needs the same type and strides", op);
    return -1;
  }
  if (n_tokens == 0) return 0;
  if (!two(op, "q_out and k_out", q_out, k_out) || !two(op, "q_out and k", q_out, k) || !two(op, "k_out and q", k_out, q)) return -1;
  const int hpw = 1024 / head_dim;
  const long long waves = (long long)n_tokens * ((n_q + n_kv + hpw - 1) / hpw), groups = (waves + 3) / 4;
  if (!grid_ok(op, groups)) return -1;
  auto go = [&](auto kern) {
    return launch(kern, groups, 256, static_cast<hipStream_t>(stream), rows_of(q), rows_of(k),
                  static_cast<const uint16_t*>(q_gain), static_cast<const uint16_t*>(k_gain), inv_freq, pos, rows_of(q_out),
                  rows_of(k_out), n_tokens, n_q, n_kv, eps);
  };
  const bool s32 = q->type == MK_TYPE_F32, d32 = q_out->type == MK_TYPE_F32;
  return launched(op, head_dim == 64 ? s32 ? (d32 ? go(norm_rope<64, true, true>) : go(norm_rope<64, true, false>))
                                           : (d32 ? go(norm_rope<64, false, true>) : go(norm_rope<64, false, false>))
                      : s32          ? (d32 ? go(norm_rope<128, true, true>) : go(norm_rope<128, true, false>))
                                     : (d32 ? go(norm_rope<128, false, true>) : go(norm_rope<128, false, false>)));
}

int megakernel_op_kv8_append(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                             const megakernel_rows* k, const megakernel_rows* v, void* stream) {
  const char* op = "op_kv8_append";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) ||
      !rows_ok(op, "k", k, cache->n_kv, cache->head_dim, false) || !rows_ok(op, "v", v, cache->n_kv, cache->head_dim, false))
    return -1;
  if (k->type != v->type) {
    set_err("%s: k and v must have one type (%d, %d)", op, k->type, v->type);
    return -1;
  }
  const int pieces = block_pieces(cache), heads = pieces < 256 ? 256 / pieces : 1;
  const long long groups = block_items(batch, cache->block) * ((cache->n_kv + heads - 1) / heads);
  if (groups == 0) return 0;
  if (!grid_ok(op, groups)) return -1;
  const bool f32 = k->type == MK_TYPE_F32;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = cache->head_dim == 64 ? launch_append<64> : launch_append<128>;
  return launched(op, go(pieces, f32, groups, st, cache_of(cache), batch_of(batch), rows_of(k), rows_of(v)));
}

int megakernel_op_kv8_read(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                           const megakernel_rows* k_out, const megakernel_rows* v_out, void* stream) {
  const char* op = "op_kv8_read";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) ||
      !rows_ok(op, "k_out", k_out, cache->n_kv, cache->head_dim, false) ||
      !rows_ok(op, "v_out", v_out, cache->n_kv, cache->head_dim, false) ||
      !apart(op, "k_out", k_out, cache->n_kv, cache->head_dim, batch->n_tokens) ||
      !apart(op, "v_out", v_out, cache->n_kv, cache->head_dim, batch->n_tokens))
    return -1;
  if (k_out->type != v_out->type) {
    set_err("%s: k_out and v_out must have one type (%d, %d)", op, k_out->type, v_out->type);
    return -1;
  }
  const long long items = block_items(batch, cache->block);
  // a piece for every thread, and several where that is more workgroups than run at once
  const bool f32 = k_out->type == MK_TYPE_F32;
  const int pieces = block_pieces(cache) * (f32 ? 2 : 1);
  int heads = pieces < 256 ? 256 / pieces : 1;
  while (heads < cache->n_kv && items * cache->n_kv > 2048ll * heads) heads *= 2;
  const long long groups = items * ((cache->n_kv + heads - 1) / heads);
  if (groups == 0) return 0;
  if (!two(op, "k_out and v_out", k_out, v_out) || !grid_ok(op, groups)) return -1;
  auto go = [&](auto kern) {
    return launch(kern, groups, 256, static_cast<hipStream_t>(stream), cache_of(cache), batch_of(batch), rows_of(k_out),
                  rows_of(v_out), heads);
  };
  return launched(op, cache->head_dim == 64 ? (f32 ? go(read_back<64, true>) : go(read_back<64, false>))
                                            : (f32 ? go(read_back<128, true>) : go(read_back<128, false>)));
}

long long megakernel_op_kv8_workspace_bytes(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch, int n_q) {
  const char* op = "op_kv8_workspace_bytes";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !heads_ok(op, n_q, cache->n_kv)) return -1;
  return workspace(plan(cache, batch, n_q), cache->n_kv, cache->head_dim);
}

int megakernel_op_kv8_attention(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                                const megakernel_rows* q, const megakernel_rows* out, int n_q, float scale,
                                void* d_workspace, long long workspace_bytes, void* stream) {
  const char* op = "op_kv8_attention";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !heads_ok(op, n_q, cache->n_kv) ||
      !rows_ok(op, "q", q, n_q, cache->head_dim, true) || !rows_ok(op, "out", out, n_q, cache->head_dim, true) ||
      !apart(op, "out", out, n_q, cache->head_dim, batch->n_tokens))
    return -1;
  if (q->p == out->p) {
    set_err("%s: out must not be q", op);
    return -1;
  }
  if ((long long)batch->n_tokens * (n_q / cache->n_kv) > (1ll << 30)) {
    set_err("%s: n_tokens=%d times %d query heads per KV head exceeds 2^30 rows", op, batch->n_tokens, n_q / cache->n_kv);
    return -1;
  }
  const float scale2 = scale * 1.4426950408889634f;  // scores are taken to base 2
  if (!(scale > 0.f && scale2 < INFINITY)) {
    set_err("%s: scale=%g must be positive and finite, also times log2(e)", op, scale);
    return -1;
  }
  const Plan pl = plan(cache, batch, n_q);
  const long long need = workspace(pl, cache->n_kv, cache->head_dim);
  if (need && (!d_workspace || !aligned(d_workspace, 16) || workspace_bytes < need)) {
    set_err("%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", op, need, d_workspace ? workspace_bytes : 0);
    return -1;
  }
  if (batch->n_tokens == 0 || batch->n_seq == 0) return 0;
  Attn p;
  p.c = cache_of(cache);
  p.b = batch_of(batch);
  p.q = rows_of(q);
  p.out = rows_of(out);
  p.n_q = n_q;
  p.group = n_q / cache->n_kv;
  p.scale = scale2;
  p.few = pl.few;
  char* ws = static_cast<char*>(d_workspace);
  for (int k = 0; k < 2; ++k) {
    Deal& d = p.d[k];
    d.lr = pl.lr[k], d.target = pl.target[k], d.least = pl.least[k], d.items = (int)pl.items[k];
    d.part = reinterpret_cast<float*>(ws);
    d.ml = reinterpret_cast<float2*>(d.part + part_floats(pl, k, cache->n_kv, cache->head_dim));
    ws += part_bytes(pl, k, cache->n_kv, cache->head_dim);
  }
  const long long few = pl.items[FEW] * cache->n_kv, many = pl.items[MANY] * cache->n_kv;
  // tokens whose rows may have splits to join
  long long tokens = batch->n_tokens;
  if (!pl.target[MANY] && pl.use[MANY] && tokens > (long long)batch->n_seq * (pl.few / p.group)) tokens = (long long)batch->n_seq * (pl.few / p.group);
  // a workgroup for every row, or where rows are many a wave for four (us in all,
  // in a graph: one row of 32,768 positions 18.9 / 31.5, 1,056 rows of drafted
  // tokens 38.8 / 40.8, a prompt's 16,384 335 / 311)
  const bool each = tokens * n_q <= 4096;
  const long long joins = !need ? 0 : each ? tokens * n_q : (tokens * ((n_q + 3) / 4) + 3) / 4;
  if (!grid_ok(op, few * 2 + many) || !grid_ok(op, joins)) return -1;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool d64 = cache->head_dim == 64;
  auto go = [&](auto kern, long long groups, int threads) { return launch(kern, groups, threads, st, p); };
  hipError_t e;
  if (pl.use[FEW] && pl.use[MANY]) e = d64 ? go(attn_both<64>, many + few, 256) : go(attn_both<128>, many + few, 256);
  else if (pl.use[MANY]) e = d64 ? go(attn_tile<64>, many, 256) : go(attn_tile<128>, many, 256);
  else if (pl.waves == 2) e = d64 ? go(attn_rows<64, 2>, few, 128) : go(attn_rows<128, 2>, few, 128);
  else if (pl.waves == 4) e = d64 ? go(attn_rows<64, 4>, few, 256) : go(attn_rows<128, 4>, few, 256);
  else e = d64 ? go(attn_rows<64, 8>, few, 512) : go(attn_rows<128, 8>, few, 512);
  if (e == hipSuccess && need) {
    if (each) e = d64 ? go(attn_join<64>, joins, 256) : go(attn_join<128>, joins, 256);
    else e = d64 ? go(attn_join_waves<64, 4>, joins, 256) : go(attn_join_waves<128, 4>, joins, 256);
  }
  return launched(op, e);
}

}  // extern "C"
