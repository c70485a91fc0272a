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

constexpr int kMaxSplits = 128;

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

static int launched(const char* op) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  set_err("%s: launch failed: %s", op, hipGetErrorString(e));
  return -1;
}

// Most workgroup items that the blocks of n_tokens rows make.
static long long block_items(const megakernel_kv8_batch* b, int block) {
  const long long n = b->n_tokens, m = n / block + 2ll * b->n_seq;
  return n < m ? n : m;
}
// Most tiles of `rows` query rows.
static long long row_tiles(const megakernel_kv8_batch* b, int group, int rows) {
  const long long n = b->n_tokens, m = n * group / rows + b->n_seq, each = n * ((group + rows - 1) / rows);
  return each < m ? each : m;
}

static int max_splits(const megakernel_kv8_cache* c, const megakernel_kv8_batch* b, int n_q) {
  const long long wg = row_tiles(b, n_q / c->n_kv, ROWS) * c->n_kv;
  if (wg < 1) return 1;
  const long long kv = b->max_kv ? b->max_kv : (long long)b->table_width * c->block;
  const long long tiles = (kv + TILE - 1) / TILE, want = (1024 + wg - 1) / wg, can = (tiles + 3) / 4;
  const long long s = want < can ? want : can;
  return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}

static long long workspace(const megakernel_kv8_cache* c, const megakernel_kv8_batch* b, int n_q) {
  const int s = max_splits(c, b, n_q);
  return s == 1 ? 0 : (long long)b->n_tokens * n_q * s * (c->head_dim + 2) * 4;
}

static bool heads_ok(const char* op, int n_q, int n_kv) {
  if (n_kv < 1 || n_kv > 1024 || n_q < 1 || n_q > 1024 || n_q % n_kv) {
    set_err("%s: n_q=%d must be a multiple of n_kv=%d (both 1..1024)", op, n_q, n_kv);
    return false;
  }
  return true;
}

template <int D>
static void launch_append(int passes, bool f32, dim3 g, hipStream_t st, Cache c, Batch b, Rows k, Rows v) {
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, g, dim3(256), 0, st, c, b, k, v); };
  if constexpr (D == 64) {
    if (passes == 1) return f32 ? go(append<D, 1, true>) : go(append<D, 1, false>);
    if (passes == 2) return f32 ? go(append<D, 2, true>) : go(append<D, 2, false>);
    return f32 ? go(append<D, 4, true>) : go(append<D, 4, false>);
  } else {
    if (passes == 1) return f32 ? go(append<D, 1, true>) : go(append<D, 1, false>);
    if (passes == 2) return f32 ? go(append<D, 2, true>) : go(append<D, 2, false>);
    if (passes == 4) return f32 ? go(append<D, 4, true>) : go(append<D, 4, false>);
    return f32 ? go(append<D, 8, true>) : go(append<D, 8, false>);
  }
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
  const int hpw = 1024 / head_dim;
  const long long waves = (long long)n_tokens * ((n_q + n_kv + hpw - 1) / hpw), groups = (waves + 3) / 4;
  if (!grid_ok(op, groups)) return -1;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, static_cast<hipStream_t>(stream), rows_of(q), rows_of(k),
                       static_cast<const uint16_t*>(q_gain), static_cast<const uint16_t*>(k_gain), inv_freq, pos,
                       rows_of(q_out), rows_of(k_out), n_tokens, n_q, n_kv, eps);
  };
  const bool s32 = q->type == MK_TYPE_F32, d32 = q_out->type == MK_TYPE_F32;
  if (head_dim == 64)
    s32 ? (d32 ? go(norm_rope<64, true, true>) : go(norm_rope<64, true, false>))
        : (d32 ? go(norm_rope<64, false, true>) : go(norm_rope<64, false, false>));
  else
    s32 ? (d32 ? go(norm_rope<128, true, true>) : go(norm_rope<128, true, false>))
        : (d32 ? go(norm_rope<128, false, true>) : go(norm_rope<128, false, false>));
  return launched(op);
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
  const long long groups = block_items(batch, cache->block) * cache->n_kv;
  if (groups == 0) return 0;
  if (!grid_ok(op, 2 * groups)) return -1;
  const dim3 g((unsigned)groups, 2);
  const int rpp = 2048 / cache->head_dim, passes = (cache->block + rpp - 1) / rpp;
  const bool f32 = k->type == MK_TYPE_F32;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 64) launch_append<64>(passes, f32, g, st, cache_of(cache), batch_of(batch), rows_of(k), rows_of(v));
  else launch_append<128>(passes, f32, g, st, cache_of(cache), batch_of(batch), rows_of(k), rows_of(v));
  return launched(op);
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
  const long long groups = block_items(batch, cache->block) * cache->n_kv;
  if (groups == 0) return 0;
  if (!grid_ok(op, 2 * groups)) return -1;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)groups, 2), dim3(256), 0, static_cast<hipStream_t>(stream), cache_of(cache),
                       batch_of(batch), rows_of(k_out), rows_of(v_out));
  };
  const bool f32 = k_out->type == MK_TYPE_F32;
  if (cache->head_dim == 64) f32 ? go(read_back<64, true>) : go(read_back<64, false>);
  else f32 ? go(read_back<128, true>) : go(read_back<128, false>);
  return launched(op);
}

long long megakernel_op_kv8_workspace_bytes(const megakernel_kv8_cache* cache, const megakernel_kv8_batch* batch, int n_q) {
  const char* op = "op_kv8_workspace_bytes";
  if (!cache_ok(op, cache) || !batch_ok(op, batch, cache->block) || !heads_ok(op, n_q, cache->n_kv)) return -1;
  return workspace(cache, batch, n_q);
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
  if (!(scale > 0.f && scale < INFINITY)) {
    set_err("%s: scale=%g must be positive and finite", op, scale);
    return -1;
  }
  const long long need = workspace(cache, batch, n_q);
  if (need && (!d_workspace || !aligned(d_workspace, 16) || workspace_bytes < need)) {
    set_err("%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", op, need, d_workspace ? workspace_bytes : 0);
    return -1;
  }
  const int group = n_q / cache->n_kv;
  const long long groups = row_tiles(batch, group, ROWS) * cache->n_kv;
  if (groups == 0) return 0;
  Attn p;
  p.c = cache_of(cache);
  p.b = batch_of(batch);
  p.q = rows_of(q);
  p.out = rows_of(out);
  p.n_q = n_q;
  p.group = group;
  p.scale = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(d_workspace);
  p.max_splits = max_splits(cache, batch, n_q);
  p.min_tiles = 4;
  if (!grid_ok(op, groups * p.max_splits)) return -1;
  const dim3 g((unsigned)groups, (unsigned)p.max_splits);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 64) hipLaunchKernelGGL(attn_rows<64>, g, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(attn_rows<128>, g, dim3(256), 0, st, p);
  if (p.max_splits > 1) {
    if (cache->head_dim == 64) hipLaunchKernelGGL(attn_join<64>, dim3((unsigned)groups), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(attn_join<128>, dim3((unsigned)groups), dim3(256), 0, st, p);
  }
  return launched(op);
}

}  // extern "C"
