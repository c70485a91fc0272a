// Host side of the paged 8-bit KV cache's operators (megakernel_op_qk_norm_rope,
// megakernel_op_rotary, megakernel_op_kv8_*): argument checks and launches.  Every call only
// enqueues on the caller's stream: no allocation, no copy, no wait, so it can
// be captured into a graph.  Lengths and block tables stay on the device; the
// grids come from the row count alone, and each workgroup finds its sequence
// there.
#include "mk_kv8.h"
#include "mk_kv8_evict.h"
#include "mk_kv8_rotary.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "megakernel.h"
#include "mk_host.h"
#include "mk_overlap.h"

namespace mk {
namespace kv8 {

static bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

static int type_size(int type) { return type == MK_TYPE_F32 ? 4 : type == MK_TYPE_BF16 ? 2 : 0; }

static bool rows_aligned(const megakernel_rows* r, int n) {
  const int sz = type_size(r->type);
  return aligned(r->p, n) && r->token_stride * sz % n == 0 && r->head_stride * sz % n == 0;
}
// A tensor of rows: type, alignment for 16-byte accesses (or, with align 0,
// that of its elements), and strides that keep the heads of one token apart.
static bool rows_ok(const char* op, const char* name, const megakernel_rows* r, int heads, int head_dim, bool bf16_only, int align = 16) {
  if (!r || !r->p) {
    set_err("%s: null %s", op, name);
    return false;
  }
  const int sz = type_size(r->type);
  if (!sz || (bf16_only && r->type != MK_TYPE_BF16)) {
    set_err("%s: %s has type %d (%s)", op, name, r->type, bf16_only ? "bf16 only" : "bf16 or fp32");
    return false;
  }
  if (!rows_aligned(r, align == 16 ? 16 : sz)) {
    set_err("%s: %s needs %d-byte aligned rows (strides %lld, %lld)", op, name, align == 16 ? 16 : sz, r->token_stride, r->head_stride);
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

static Span span_of(const megakernel_rows* r, long long tokens, int heads, long long head_dim) {
  const int sz = type_size(r->type);
  return Span{(uintptr_t)r->p, tokens, heads, r->token_stride * sz, r->head_stride * sz, head_dim * sz};
}
static Span span_of(const void* words, long long n) { return Span{(uintptr_t)words, 1, 1, 0, 0, 4 * n}; }  // int or fp32

// Two tensors, one of them written, that cannot be the same or lie on each other.
static bool two(const char* op, const char* names, const Span& a, const Span& b) {
  if (a.p != b.p && !overlap(a, b)) return true;
  set_err("%s: %s must not be the same rows, or lie on each other", op, names);
  return false;
}

// Queries and keys that are turned: one type in and one out, and outputs in
// place of inputs only where a lane writes what it alone has read.
static bool turned_ok(const char* op, const megakernel_rows* q, const megakernel_rows* k, const megakernel_rows* q_out,
                      const megakernel_rows* k_out, int n_tokens, int n_q, int n_kv, int head_dim) {
  if (q->type != k->type || q_out->type != k_out->type) {
    set_err("%s: q and k must have one type (%d, %d), and so must q_out and k_out (%d, %d)", op, q->type, k->type,
            q_out->type, k_out->type);
    return false;
  }
  const Span sq = span_of(q, n_tokens, n_q, head_dim), sk = span_of(k, n_tokens, n_kv, head_dim);
  const Span dq = span_of(q_out, n_tokens, n_q, head_dim), dk = span_of(k_out, n_tokens, n_kv, head_dim);
  auto moved = [](const megakernel_rows* a, const megakernel_rows* b, const Span& x, const Span& y) {
    if (a->p != b->p) return overlap(x, y);
    return a->type != b->type || a->token_stride != b->token_stride || a->head_stride != b->head_stride;
  };
  if (moved(q, q_out, sq, dq) || moved(k, k_out, sk, dk)) {
    set_err("%s: an output in place of its input needs the same start, type and strides", op);
    return false;
  }
  return n_tokens == 0 || (two(op, "q_out and k_out", dq, dk) && two(op, "q_out and k", dq, sk) && two(op, "k_out and q", dk, sq));
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
static Plan plan(const megakernel_kv8_cache* c, const megakernel_kv8_batch* b, int n_q, const megakernel_kv8_scores* x = nullptr) {
  Plan p{};
  const int group = n_q / c->n_kv;
  const bool d64 = c->head_dim == 64;
  const int window = x ? x->window : 0;
  const long long rows = (long long)b->n_tokens * group;
  long long kv = b->max_kv ? b->max_kv : (long long)b->table_width * c->block;
  if (window && kv > (long long)window + TILE) kv = (long long)window + TILE;  // a window lies across one step more
  const long long steps = (kv + TILE - 1) / TILE;
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
      // 19 / 13 / 15, of 64 53 / 50 / 52; 4,096 of 1 50 / 25 / 18).  With scores the
      // kernels hold 135 registers and more, three waves a SIMD: of eight waves one
      // workgroup fits a CU, of four three, so from a workgroup a CU on it is four
      // (capped, head_dim 64, 8 / 4 waves; 264 workgroups of 64 steps 36 / 30, 320 of
      // 50 30 / 27, of 64 37 / 32, of 128 73 / 64, 512 of 64 44.5 / 43.9; 128: 68 / 66,
      // 54 / 52, 73 / 71, 144 / 144, 95 / 94).
      const long long low = (rows / ROWS > b->n_seq ? rows / ROWS : b->n_seq) * c->n_kv;
      p.waves = low >= 1024 ? (steps <= 8 ? 2 : 4) : (x && low > 256) || steps <= (low > 256 ? 48 : 8) ? 4 : 8;
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
static long long part_rows(const Plan& p, int k, int n_kv) { return p.slots[k] * n_kv << p.lr[k]; }
static long long part_bytes(const Plan& p, int k, int n_kv, int head_dim) {
  return part_floats(p, k, n_kv, head_dim) * 4 + part_rows(p, k, n_kv) * 8;
}
// `lse`: with the sums of the weights before their rounding, behind the rest
static long long workspace(const Plan& p, int n_kv, int head_dim, bool lse) {
  return part_bytes(p, FEW, n_kv, head_dim) + part_bytes(p, MANY, n_kv, head_dim) +
         (lse ? 4 * (part_rows(p, FEW, n_kv) + part_rows(p, MANY, n_kv)) : 0);
}

// Tokens whose rows may have splits to join.
static long long joined_tokens(const Plan& p, const megakernel_kv8_batch* b, int group) {
  const long long few = (long long)b->n_seq * (p.few / group);
  return !p.target[MANY] && p.use[MANY] && b->n_tokens > few ? few : b->n_tokens;
}
// A workgroup for every row, or where rows are many a wave for four (us in all,
// in a graph: one row of 32,768 positions 18.9 / 31.5, 1,056 rows of drafted
// tokens 38.8 / 40.8, a prompt's 16,384 335 / 311).
static bool join_each(long long tokens, int n_q) { return tokens * n_q <= 4096; }

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

static bool scores_ok(const char* op, const megakernel_kv8_scores* x) {
  if (!x) {
    set_err("%s: null scores", op);
    return false;
  }
  if (!aligned(x->slopes, 4) || !aligned(x->first, 4) || !aligned(x->prefix, 4)) {
    set_err("%s: slopes, first and prefix need 4-byte alignment", op);
    return false;
  }
  if (!(x->softcap == 0.f || (x->softcap >= 0x1p-30f && x->softcap <= 1024.f)) || x->window < 0) {
    set_err("%s: softcap=%g (0, or 2^-30 to 1024), window=%d (0, or at least 1)", op, x->softcap, x->window);
    return false;
  }
  return true;
}

// The softmax scale to base 2, or 0 where it cannot be.
static float scale_of(const char* op, const megakernel_kv8_scores* x, float scale) {
  const float scale2 = scale * 1.4426950408889634f;  // scores are taken to base 2
  if (!(scale > 0.f && scale2 < INFINITY)) {
    set_err("%s: scale=%g must be positive and finite, also times log2(e)", op, scale);
    return 0.f;
  }
  if (x && x->softcap > 0.f && !(scale2 / x->softcap >= 0x1p-120f && scale2 / x->softcap <= 0x1p120f)) {
    set_err("%s: scale=%g is too far from softcap=%g", op, scale, x->softcap);
    return 0.f;
  }
  return scale2;
}
static Scores scores_of(const megakernel_kv8_scores* x, float scale2) {
  Scores r{x->slopes, x->first, x->prefix, x->window, 0.f, 0.f, {}};
  if (x->softcap > 0.f) {
    r.cap = x->softcap * 1.4426950408889634f;
    r.cap_in = scale2 / r.cap;
    // (tanh(sqrt(w)) / sqrt(w) - 1) / w at Chebyshev's nodes of [0, 1/4]
    const float q[4] = {-0x1.555546p-2f, 0x1.110246p-3f, -0x1.b560bap-5f, 0x1.26e43ep-6f};
    for (int i = 0; i < 4; ++i) r.c[i] = r.cap * q[i];
  }
  return r;
}

// P: Attn, AttnScored with x, or AttnLse with x and lse.
template <class P>
static int attend(const char* op, const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                  const megakernel_kv8_scores* x, const megakernel_rows* q, const megakernel_rows* out, float* lse, int n_q,
                  float scale, void* d_workspace, long long workspace_bytes, hipStream_t st) {
  constexpr bool SCORED = Has<P>::scores, LSE = Has<P>::lse;
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !heads_ok(op, n_q, cache->n_kv) ||
      !rows_ok(op, "q", q, n_q, cache->head_dim, true) || !rows_ok(op, "out", out, n_q, cache->head_dim, true) ||
      !apart(op, "out", out, n_q, cache->head_dim, batch->n_tokens) || (SCORED && !scores_ok(op, x)))
    return -1;
  if (!aligned(lse, 4)) {
    set_err("%s: lse needs 4-byte alignment", op);
    return -1;
  }
  if (q->p == out->p) {
    set_err("%s: out must not be q", op);
    return -1;
  }
  if ((long long)batch->n_tokens * (n_q / cache->n_kv) > (1ll << 30)) {
    set_err("%s: n_tokens=%d times %d query heads per KV head exceeds 2^30 rows", op, batch->n_tokens, n_q / cache->n_kv);
    return -1;
  }
  const float scale2 = scale_of(op, x, scale);
  if (!scale2) return -1;
  const Plan pl = plan(cache, batch, n_q, x);
  const long long need = workspace(pl, cache->n_kv, cache->head_dim, LSE);
  if (need && (!d_workspace || !aligned(d_workspace, 16) || workspace_bytes < need)) {
    set_err("%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", op, need, d_workspace ? workspace_bytes : 0);
    return -1;
  }
  if (batch->n_tokens == 0 || batch->n_seq == 0) return 0;
  const Span sq = span_of(q, batch->n_tokens, n_q, cache->head_dim), so = span_of(out, batch->n_tokens, n_q, cache->head_dim);
  const Span sl = span_of(lse, (long long)batch->n_tokens * n_q);
  if (!two(op, "out and q", so, sq)) return -1;
  if (LSE && (!two(op, "lse and q", sl, sq) || !two(op, "lse and out", sl, so))) return -1;
  P p;
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
  if constexpr (SCORED) p.x = scores_of(x, scale2);
  if constexpr (LSE) {
    p.lse = lse;
    p.ex[FEW] = reinterpret_cast<float*>(ws);
    p.ex[MANY] = p.ex[FEW] + part_rows(pl, FEW, cache->n_kv);
  }
  const long long few = pl.items[FEW] * cache->n_kv, many = pl.items[MANY] * cache->n_kv;
  const long long tokens = joined_tokens(pl, batch, p.group);
  const bool each = join_each(tokens, n_q);
  const long long joins = !need ? 0 : each ? tokens * n_q : (tokens * ((n_q + 3) / 4) + 3) / 4;
  if (!grid_ok(op, few * 2 + many) || !grid_ok(op, joins)) return -1;
  const bool d64 = cache->head_dim == 64;
  auto go = [&](auto kern, long long groups, int threads) { return launch(kern, groups, threads, st, p); };
  hipError_t e;
  if (pl.use[FEW] && pl.use[MANY]) e = d64 ? go(attn_both<64, P>, many + few, 256) : go(attn_both<128, P>, many + few, 256);
  else if (pl.use[MANY]) e = d64 ? go(attn_tile<64, P>, many, 256) : go(attn_tile<128, P>, many, 256);
  else if (pl.waves == 2) e = d64 ? go(attn_rows<64, 2, P>, few, 128) : go(attn_rows<128, 2, P>, few, 128);
  else if (pl.waves == 4) e = d64 ? go(attn_rows<64, 4, P>, few, 256) : go(attn_rows<128, 4, P>, few, 256);
  else e = d64 ? go(attn_rows<64, 8, P>, few, 512) : go(attn_rows<128, 8, P>, few, 512);
  if (e == hipSuccess && need) {
    if (each) e = d64 ? go(attn_join<64, P>, joins, 256) : go(attn_join<128, P>, joins, 256);
    else e = d64 ? go(attn_join_waves<64, 4, P>, joins, 256) : go(attn_join_waves<128, 4, P>, joins, 256);
  }
  return launched(op, e);
}

// Weights of cached positions: fp32 rows [n_seq][n_kv] of all positions that a table holds.
static bool mass_ok(const char* op, const char* name, const megakernel_rows* m, int n_seq, int n_kv, long long positions) {
  if (!rows_ok(op, name, m, n_kv, (int)positions, false, 0) || !apart(op, name, m, n_kv, (int)positions, n_seq)) return false;
  if (m->type == MK_TYPE_F32) return true;
  set_err("%s: %s must be fp32", op, name);
  return false;
}
static Mass mass_of(const megakernel_rows* m) { return Mass{static_cast<float*>(m->p), m->token_stride, m->head_stride}; }

template <int D>
static hipError_t launch_move(int pieces, long long groups, hipStream_t st, const Move& p) {
  auto go = [&](auto kern) { return launch(kern, groups, 256, st, p); };
  if constexpr (D == 64)
    if (pieces == 64) return go(move<D, 64, 1>);
  if (pieces == 128) return go(move<D, 128, 1>);
  if (pieces == 512) return go(move<D, 256, 2>);
  if constexpr (D == 128)
    if (pieces == 1024) return go(move<D, 256, 4>);
  return go(move<D, 256, 1>);
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
  if (!turned_ok(op, q, k, q_out, k_out, n_tokens, n_q, n_kv, head_dim)) return -1;
  if (n_tokens == 0) return 0;
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
  const Span sk = span_of(k_out, batch->n_tokens, cache->n_kv, cache->head_dim);
  if (!two(op, "k_out and v_out", sk, span_of(v_out, batch->n_tokens, cache->n_kv, cache->head_dim)) || !grid_ok(op, groups)) return -1;
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
  return workspace(plan(cache, batch, n_q), cache->n_kv, cache->head_dim, false);
}

int megakernel_op_kv8_attention(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                                const megakernel_rows* q, const megakernel_rows* out, int n_q, float scale,
                                void* d_workspace, long long workspace_bytes, void* stream) {
  return attend<Attn>("op_kv8_attention", cache, batch, nullptr, q, out, nullptr, n_q, scale, d_workspace, workspace_bytes,
                      static_cast<hipStream_t>(stream));
}

long long megakernel_op_kv8_scored_workspace_bytes(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                                                   const megakernel_kv8_scores* scores, int n_q, int with_lse) {
  const char* op = "op_kv8_scored_workspace_bytes";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !scores_ok(op, scores) || !heads_ok(op, n_q, cache->n_kv)) return -1;
  return workspace(plan(cache, batch, n_q, scores), cache->n_kv, cache->head_dim, with_lse != 0);
}

int megakernel_op_kv8_attention_scored(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                                       const megakernel_kv8_scores* scores, const megakernel_rows* q,
                                       const megakernel_rows* out, float* lse, int n_q, float scale, void* d_workspace,
                                       long long workspace_bytes, void* stream) {
  const auto go = lse ? attend<AttnLse> : attend<AttnScored>;
  return go("op_kv8_attention_scored", cache, batch, scores, q, out, lse, n_q, scale, d_workspace, workspace_bytes,
            static_cast<hipStream_t>(stream));
}

int megakernel_op_kv8_attention_kernels(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                                        const megakernel_kv8_scores* scores, int n_q) {
  const char* op = "op_kv8_attention_kernels";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || (scores && !scores_ok(op, scores)) || !heads_ok(op, n_q, cache->n_kv)) return -1;
  const Plan p = plan(cache, batch, n_q, scores);
  int r = 0;
  if (p.use[FEW]) r |= MK_KV8_ROWS | (p.target[FEW] ? MK_KV8_ROWS_SPLIT : 0);
  if (p.use[MANY]) r |= MK_KV8_TILE | (p.target[MANY] ? MK_KV8_TILE_SPLIT : 0);
  if ((p.target[FEW] || p.target[MANY]) && !join_each(joined_tokens(p, batch, n_q / cache->n_kv), n_q)) r |= MK_KV8_JOIN_WAVES;
  return r;
}

int megakernel_op_kv8_weigh(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch,
                            const megakernel_kv8_scores* scores, const megakernel_rows* q, const float* lse,
                            const megakernel_rows* mass, int n_q, float scale, void* stream) {
  const char* op = "op_kv8_weigh";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !scores_ok(op, scores) || !heads_ok(op, n_q, cache->n_kv) ||
      !rows_ok(op, "q", q, n_q, cache->head_dim, true) ||
      !mass_ok(op, "mass", mass, batch->n_seq, cache->n_kv, (long long)batch->table_width * cache->block))
    return -1;
  if (!lse || !aligned(lse, 4)) {
    set_err("%s: null lse, or not 4-byte aligned", op);
    return -1;
  }
  const int group = n_q / cache->n_kv;
  const long long rows = (long long)batch->n_tokens * group, all = (long long)batch->table_width * cache->block;
  if (rows > (1ll << 30) || batch->n_seq * ((all + 31) / 32) > (1ll << 30)) {
    set_err("%s: n_tokens=%d times %d query heads per KV head exceeds 2^30 rows, or n_seq=%d times %lld positions 2^35", op,
            batch->n_tokens, group, batch->n_seq, all);
    return -1;
  }
  const float scale2 = scale_of(op, scores, scale);
  if (!scale2) return -1;
  if (batch->n_tokens == 0 || batch->n_seq == 0) return 0;
  const Span sm = span_of(mass, batch->n_seq, cache->n_kv, all);
  if (!two(op, "mass and lse", sm, span_of(lse, (long long)batch->n_tokens * n_q)) ||
      !two(op, "mass and q", sm, span_of(q, batch->n_tokens, n_q, cache->head_dim)))
    return -1;
  Weigh p{cache_of(cache), batch_of(batch), rows_of(q), lse, mass_of(mass), n_q, group, scale2, scores_of(scores, scale2)};
  long long kv = batch->max_kv && batch->max_kv < all ? batch->max_kv : all;
  const long long steps = (kv + TILE - 1) / TILE * batch->n_seq, items = steps * cache->n_kv;
  // Of weigh_many in steps of 32 positions where those of 64 are not two workgroups
  // for every CU (1,024 tokens in steps of 32 / 64, head_dim 128: at 1,024 positions
  // 13 / 20, 2,048 21 / 22, 4,096 39 / 34, 8,192 72 / 64).
  const bool small = items < 512;
  // Steps of 64 positions: a wave's with few rows, a workgroup's with many.  512 such
  // workgroups run at once and take 4 us and more to start, a wave is long at many
  // rows: where one round of workgroups is all, they pay from 80 rows a sequence on,
  // else from as many as a third of the steps, until the waves' own way is bound by
  // its operations (us of weigh_few / weigh_many, 16 / 8 heads; head_dim 64, one
  // sequence of 1,024 positions, 32 rows 6.4 / 6.6, 64 8.0 / 6.5; of 4,096, 64 rows
  // 8.0 / 8.3, 128 11.2 / 9.1; of 8,192, 320 rows 17.1 / 17.6, 384 20.5 / 18.7; three
  // of 1,024, 128 rows 11.2 / 11.1; 16 of 1,024, 512 rows 29 / 37, 1,024 51 / 52; 8 of
  // 4,096, 1,024 rows 91 / 99, 1,536 133 / 129; 16 of 4,096, 1,024 rows 178 / 182, 1,536
  // 262 / 239; 128: one of 4,096, 64 rows 9.5 / 9.5, 128 13.0 / 10.2; of 8,192, 320 rows
  // 20.5 / 21.3, 384 24.3 / 22.9; 8 of 4,096, 320 rows 70 / 73, 512 105 / 93; 16 of 4,096,
  // 384 rows 133 / 143, 512 172 / 168).
  const long long most = (small ? 2 * items : items) <= 512 ? 80 : cache->head_dim == 64 ? 1280 : 512;
  const long long enough = items / 3 < 32 ? 32 : items / 3 > most ? most : items / 3;
  const bool many = rows > enough * batch->n_seq, half = many && small;
  long long groups = half ? 2 * steps : many ? steps : (steps + 3) / 4;
  // more than one step each where that is more workgroups than run at once
  if (groups > 4096 / cache->n_kv) groups = 4096 / cache->n_kv;
  groups = (groups < 1 ? 1 : groups) * cache->n_kv;
  auto go = [&](auto kern, int threads) { return launch(kern, groups, threads, static_cast<hipStream_t>(stream), p); };
  if (!many) return launched(op, cache->head_dim == 64 ? go(weigh_few<64>, 256) : go(weigh_few<128>, 256));
  return launched(op, cache->head_dim == 64 ? (half ? go(weigh_many<64, 1>, 512) : go(weigh_many<64, 2>, 512))
                                            : (half ? go(weigh_many<128, 1>, 512) : go(weigh_many<128, 2>, 512)));
}

int megakernel_op_kv8_select(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch, const megakernel_rows* mass,
                             int keep, int recent, int sinks, int* kept, int* kept_len, void* stream) {
  const char* op = "op_kv8_select";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block)) return -1;
  const long long all = (long long)batch->table_width * cache->block;
  if (!mass_ok(op, "mass", mass, batch->n_seq, cache->n_kv, all)) return -1;
  if (keep < 1 || keep > (1 << 30) || recent < 0 || sinks < 0 || (long long)recent + sinks > keep) {
    set_err("%s: keep=%d (1..2^30), recent=%d and sinks=%d (at least 0, together at most keep)", op, keep, recent, sinks);
    return -1;
  }
  if (!kept || !kept_len || !aligned(kept, 4) || !aligned(kept_len, 4)) {
    set_err("%s: null kept or kept_len, or not 4-byte aligned", op);
    return -1;
  }
  const Span sl = span_of(kept_len, batch->n_seq), sk = span_of(kept, (long long)batch->n_seq * cache->n_kv * keep);
  const Span from = span_of(batch->kv_len, batch->n_seq), sm = span_of(mass, batch->n_seq, cache->n_kv, all);
  if (kept_len == batch->kv_len || overlap(sl, from)) {  // heads would read what others have written
    set_err("%s: kept_len must not be kv_len, or lie on it", op);
    return -1;
  }
  if (batch->n_seq == 0) return 0;
  if (!two(op, "kept and kv_len", sk, from) || !two(op, "kept and kept_len", sk, sl) || !two(op, "kept and mass", sk, sm) ||
      !two(op, "kept_len and mass", sl, sm))
    return -1;
  const long long groups = (long long)batch->n_seq * cache->n_kv;
  if (!grid_ok(op, groups * 4)) return -1;
  Choose p{mass_of(mass), batch->kv_len, kept, kept_len, cache->n_kv, keep, recent, sinks, (int)all};
  const long long kv = batch->max_kv && batch->max_kv < all ? batch->max_kv : all, most = kv - recent - sinks;
  auto go = [&](auto kern) { return launch(kern, groups, 1024, static_cast<hipStream_t>(stream), p); };
  // so much LDS that two workgroups share a CU, or that 32,768 weights stay in it
  return launched(op, most <= 4096 ? go(choose<4>) : go(choose<32>));
}

int megakernel_op_kv8_compact(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch, const int* kept,
                              const int* kept_len, int keep, const int* new_table, int new_width, const megakernel_rows* mass,
                              const megakernel_rows* new_mass, void* stream) {
  const char* op = "op_kv8_compact";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block)) return -1;
  if (!kept || !kept_len || !new_table || !aligned(kept, 4) || !aligned(kept_len, 4) || !aligned(new_table, 4)) {
    set_err("%s: null kept, kept_len or new_table, or not 4-byte aligned", op);
    return -1;
  }
  const long long all = (long long)batch->table_width * cache->block, room = (long long)new_width * cache->block;
  if (keep < 1 || keep > (1 << 30) || new_width < 1 || room > (1ll << 30)) {
    set_err("%s: keep=%d (1..2^30), new_width=%d blocks of %d positions (at least 1 block, at most 2^30 positions)", op, keep,
            new_width, cache->block);
    return -1;
  }
  const Span fresh = span_of(new_table, (long long)batch->n_seq * new_width);
  if (new_table == batch->table || overlap(fresh, span_of(batch->table, (long long)batch->n_seq * batch->table_width))) {
    set_err("%s: new_table must not be the batch's table, or lie on it: rows would go where others are read", op);
    return -1;
  }
  if (!mass != !new_mass) {
    set_err("%s: mass and new_mass go together", op);
    return -1;
  }
  if (mass && (!mass_ok(op, "mass", mass, batch->n_seq, cache->n_kv, all) ||
               !mass_ok(op, "new_mass", new_mass, batch->n_seq, cache->n_kv, room)))
    return -1;
  if (mass) {
    const Span to = span_of(new_mass, batch->n_seq, cache->n_kv, room);
    if (!two(op, "mass and new_mass", span_of(mass, batch->n_seq, cache->n_kv, all), to) || !two(op, "new_mass and new_table", to, fresh) ||
        !two(op, "new_mass and kept", to, span_of(kept, (long long)batch->n_seq * cache->n_kv * keep)) ||
        !two(op, "new_mass and kept_len", to, span_of(kept_len, batch->n_seq)))
      return -1;
  }
  if (batch->n_seq == 0) return 0;
  const int pieces = cache->block * cache->head_dim / 16, heads = pieces < 256 ? 256 / pieces : 1;
  const long long per = ((long long)keep + cache->block - 1) / cache->block;
  const long long groups = batch->n_seq * per * ((cache->n_kv + heads - 1) / heads);
  if (!grid_ok(op, groups)) return -1;
  Move p{cache_of(cache), batch->table, kept, kept_len, new_table, batch->table_width, new_width, keep, Mass{}, Mass{}};
  if (mass) p.from = mass_of(mass), p.to = mass_of(new_mass);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return launched(op, cache->head_dim == 64 ? launch_move<64>(pieces, groups, st, p) : launch_move<128>(pieces, groups, st, p));
}

int megakernel_op_rotary(const megakernel_rows* q, const megakernel_rows* k, const float* inv_freq, const int* pos,
                         const megakernel_rows* q_out, const megakernel_rows* k_out, int n_tokens, int n_q, int n_kv,
                         int head_dim, int turned, int interleaved, float amplitude, void* stream) {
  const char* op = "op_rotary";
  if (head_dim < 2 || head_dim > 1024 || head_dim % 2 || turned < 2 || turned > head_dim || turned % 2) {
    set_err("%s: head_dim=%d (even, 2..1024), turned=%d (even, 2..head_dim)", op, head_dim, turned);
    return -1;
  }
  if (n_q < 1 || n_q > 1024 || n_kv < 1 || n_kv > 1024 || n_tokens < 0 || n_tokens > (1 << 27)) {
    set_err("%s: n_q=%d, n_kv=%d (both 1..1024), n_tokens=%d (0..2^27)", op, n_q, n_kv, n_tokens);
    return -1;
  }
  if (!(fabsf(amplitude) < INFINITY)) {
    set_err("%s: amplitude=%g must be finite", op, amplitude);
    return -1;
  }
  if (!rows_ok(op, "q", q, n_q, head_dim, false, 0) || !rows_ok(op, "k", k, n_kv, head_dim, false, 0) ||
      !rows_ok(op, "q_out", q_out, n_q, head_dim, false, 0) || !rows_ok(op, "k_out", k_out, n_kv, head_dim, false, 0) ||
      !apart(op, "q_out", q_out, n_q, head_dim, n_tokens) || !apart(op, "k_out", k_out, n_kv, head_dim, n_tokens))
    return -1;
  if (!inv_freq || !pos || !aligned(inv_freq, 4) || !aligned(pos, 4)) {
    set_err("%s: null or unaligned inv_freq or pos (4 bytes)", op);
    return -1;
  }
  if (!turned_ok(op, q, k, q_out, k_out, n_tokens, n_q, n_kv, head_dim)) return -1;
  if (n_tokens == 0) return 0;
  const Turn p{rows_of(q), rows_of(k), rows_of(q_out), rows_of(k_out), inv_freq, pos, n_tokens, n_q, n_kv, head_dim, turned, amplitude};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool s32 = q->type == MK_TYPE_F32, d32 = q_out->type == MK_TYPE_F32;
  long long groups;
  auto go = [&](auto kern, auto... more) { return launch(kern, groups, 256, st, p, more...); };
  if (head_dim % 16 || turned % 16 || !rows_aligned(q, 16) || !rows_aligned(k, 16) || !rows_aligned(q_out, 16) || !rows_aligned(k_out, 16)) {
    groups = ((long long)n_tokens * (n_q + n_kv) * (head_dim / 2) + 255) / 256;
    if (!grid_ok(op, groups)) return -1;
    return launched(op, s32 ? (d32 ? go(rotate_pairs<true, true>, interleaved) : go(rotate_pairs<true, false>, interleaved))
                            : (d32 ? go(rotate_pairs<false, true>, interleaved) : go(rotate_pairs<false, false>, interleaved)));
  }
  const long long units = (long long)n_tokens * (head_dim / 16);
  // four heads share a set of sines where that still fills the chip (us with one /
  // four, 24 heads of 128, bf16: 512 tokens 3.7 / 4.1, 1,024 4.75 / 4.6, 4,096 14.5 / 10.1)
  const bool many = units * (n_q + n_kv) > 1 << 17;
  groups = (units * (many ? (n_q + n_kv + 3) / 4 : n_q + n_kv) + 255) / 256;
  if (!grid_ok(op, groups)) return -1;
  auto pick = [&](auto il, auto n) {
    constexpr bool I = decltype(il)::value;
    constexpr int N = decltype(n)::value;
    return s32 ? (d32 ? go(rotate<true, true, I, N>) : go(rotate<true, false, I, N>))
               : (d32 ? go(rotate<false, true, I, N>) : go(rotate<false, false, I, N>));
  };
  return launched(op, interleaved ? (many ? pick(Bool<true>{}, Int<4>{}) : pick(Bool<true>{}, Int<1>{}))
                                  : (many ? pick(Bool<false>{}, Int<4>{}) : pick(Bool<false>{}, Int<1>{})));
}

}  // extern "C"
