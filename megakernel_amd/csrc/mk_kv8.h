// Kernels of the paged 8-bit KV cache's operators (kv8.hip has their host
// side).  The cache is a pool of blocks of B positions (16, 32, 64 or 128):
//   K codes  [n_blocks][n_kv][B][D]   one position's row contiguous
//   V codes  [n_blocks][n_kv][D][B]   one dimension's positions contiguous
//   scales   [n_blocks][n_kv] fp32    one power of two for K, one for V
// Codes are OCP e4m3, value = code * scale.  A sequence's block table names
// its blocks in order; entries outside [0, n_blocks) are missing blocks.
//
// Power-of-two scales: dividing by one and multiplying by it are exact, a
// code times its scale is exact in bf16, and a scale can grow (a partly
// filled block takes a larger row) by re-rounding codes alone.  V lies
// transposed so that both products of the attention take cache bytes as the
// A operand of v_mfma_f32_16x16x32_bf16 straight from 16-byte loads.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "megakernel.h"
#include "mk_device.h"

namespace mk {
namespace kv8 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int n_blocks, n_kv, lb;  // lb: log2 of the positions per block
};

struct Batch {
  const int* table;
  const int* start;
  const int* len;
  int n_seq, width, n_tokens;
};

struct Rows {
  void* p;
  long long ts, hs;  // elements from one token / head to the next
};

// One sequence's rows: first row, rows, and the position of the first one
// (negative where more rows than positions were given).
struct Seq {
  int i, row0, rows, pos0, len;
};

// Sequence i, with every value brought into the buffers' bounds: row numbers
// into [0, n_tokens], the length into [0, positions of the table].  pos0
// follows from the length as given, so a row keeps its own position.
__device__ __forceinline__ Seq seq_at(const Batch& b, int i, int lb) {
  Seq s;
  s.i = i;
  const int a = b.start[i], e = b.start[i + 1], l = b.len[i];
  const int a0 = min(max(a, 0), b.n_tokens);
  s.row0 = a0;
  s.rows = max(min(max(e, 0), b.n_tokens) - a0, 0);
  // a row's position counts back from the length; saturated, so that no
  // garbage in `start` wraps it
  const long long p = (long long)l - ((long long)e - a0);
  s.pos0 = (int)max(min(p, 0x7fffff00ll - s.rows), -0x7fffff00ll);
  s.len = min(max(l, 0), b.width << lb);
  return s;
}

// Work items are dealt to the sequences in order, count(seq) each; finds the
// sequence of item `it` and the item's number within it.  A wave looks at 64
// sequences at a time (the whole wave must call it).  False past the last.
template <class Count>
__device__ __forceinline__ bool find_item(const Batch& b, int lb, int it, Count count, Seq& s, int& within) {
  const int l = (int)(threadIdx.x & (kWave - 1u));
  int before = 0;
  for (int base = 0; base < b.n_seq; base += kWave) {
    int c = 0;
    if (base + l < b.n_seq) c = count(seq_at(b, base + l, lb));
    int sum = c;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (l >= d) sum += o;
    }
    const unsigned long long hit = __ballot(before + sum > it);
    if (hit) {
      const int f = __ffsll((long long)hit) - 1;
      within = it - before - (__shfl(sum, f) - __shfl(c, f));
      s = seq_at(b, __builtin_amdgcn_readfirstlane(base + f), lb);
      within = __builtin_amdgcn_readfirstlane(within);
      return true;
    }
    before += __shfl(sum, kWave - 1);
  }
  return false;
}

// Blocks that a sequence's rows lie in.
__device__ __forceinline__ int blocks_touched(const Seq& s, int lb) {
  const int p0 = max(s.pos0, 0), p1 = min(s.pos0 + s.rows, s.len);  // written or read positions
  return p1 > p0 ? ((p1 - 1) >> lb) - (p0 >> lb) + 1 : 0;
}

// Block of position block number j of sequence i, or -1.
__device__ __forceinline__ int block_id(const Batch& b, int i, int j, int n_blocks) {
  if (j < 0 || j >= b.width) return -1;
  const int id = b.table[(long long)i * b.width + j];
  return id >= 0 && id < n_blocks ? id : -1;
}

// Eight consecutive elements of a row as fp32, and back.
template <bool F32>
__device__ __forceinline__ void load8(const void* p, long long e, float (&f)[8]) {
  if constexpr (F32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + e);
    const float4 a = q[0], b = q[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
  }
}
template <bool F32>
__device__ __forceinline__ void store8(void* p, long long e, const float (&f)[8]) {
  if constexpr (F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + e);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f[2 * i], f[2 * i + 1]}, bf16x2));
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + e) = w;
  }
}

// ------------------------------------------------- norms with the rotation
// y = x * rsqrt(mean(x^2) + eps) * gain over a head, then for each pair
// (i, i + D/2) the rotation by pos * inv_freq[i].  A head takes D/16 lanes:
// lane j holds elements 8j..8j+7 of both halves, so a pair never leaves its
// lane and the mean is a DPP sum.  The angle is a product of a 24-bit and a
// 31-bit number, formed and reduced to a fraction of a turn in fp64 (fp32
// would be off by 2^-24 of an angle of up to 1e5 radians); the sine and
// cosine of the fraction are fp32.
template <int D, bool SRC32, bool DST32>
__global__ __launch_bounds__(256) void norm_rope(Rows q, Rows k, const uint16_t* __restrict__ qg,
                                                 const uint16_t* __restrict__ kg, const float* __restrict__ freq,
                                                 const int* __restrict__ pos, Rows qo, Rows ko, int n_tokens, int n_q,
                                                 int n_kv, float eps) {
  constexpr int LPH = D / 16, HPW = kWave / LPH;  // lanes per head, heads per wave
  const int l = (int)(threadIdx.x & 63u), j = l % LPH;
  const int heads = n_q + n_kv, passes = (heads + HPW - 1) / HPW;
  const long long it = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  const int t = (int)(it / passes), h = (int)(it % passes) * HPW + l / LPH;
  if (t >= n_tokens || h >= heads) return;
  const bool is_k = h >= n_q;
  const Rows& src = is_k ? k : q;
  const Rows& dst = is_k ? ko : qo;
  const int hh = is_k ? h - n_q : h;
  float a[8], b[8], ga[8], gb[8];
  const long long e = t * src.ts + hh * src.hs + 8 * j;
  load8<SRC32>(src.p, e, a);
  load8<SRC32>(src.p, e + D / 2, b);
  const uint16_t* g = is_k ? kg : qg;
  load8<false>(g, 8 * j, ga);
  load8<false>(g, 8 * j + D / 2, gb);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
  ss = group_sum<LPH>(ss);
  const float r = rsqrtf(ss * (1.f / D) + eps);
  const double p = (double)pos[t] * 0.15915494309189535;  // turns of one radian
  float oa[8], ob[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double turns = p * (double)freq[8 * j + i];
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * (float)turns, &sn, &cs);
    const float x = a[i] * r * ga[i], y = b[i] * r * gb[i];
    oa[i] = x * cs - y * sn;
    ob[i] = y * cs + x * sn;
  }
  const long long o = t * dst.ts + hh * dst.hs + 8 * j;
  store8<DST32>(dst.p, o, oa);
  store8<DST32>(dst.p, o + D / 2, ob);
}

// ------------------------------------------------------- quantised append
// Exponent of the smallest power of two s >= 2^-126 with amax <= 448 s
// (448 = 1.75 * 2^8).  Zero rows give 2^-126, so that a block that starts
// with them takes the scale of the rows that follow.
__device__ __forceinline__ int scale_exp(float amax) {
  if (!(amax > 0.f)) return -126;
  int e = ilogbf(amax) - 8;
  if (amax > ldexpf(448.f, e)) ++e;
  return max(e, -126);
}

// Codes of four values that were divided by the scale: nearest, ties to even;
// beyond 448 (infinities alone) saturated; NaN stays NaN.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const auto cl = [](float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); };
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(a), cl(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(c), cl(d), w, true);
  return (uint32_t)w;
}
// Four codes re-rounded after multiplying by a power of two of at most one.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return encode4(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}

// x * 2^-e for e in [-126, 120], exactly: two factors where one would leave
// fp32's range.
struct Unscale {
  float f, g;
};
__device__ __forceinline__ Unscale unscale(int e) {
  const int h = -e / 2;
  return Unscale{ldexpf(1.f, h), ldexpf(1.f, -e - h)};
}

// One workgroup per (block that rows go to, head, K or V).  A thread holds 8
// dimensions of one row per pass; all rows of the block stay in registers
// between the maximum and the rounding, so the input is read once.
template <int D, int PASSES, bool SRC32>
__global__ __launch_bounds__(256) void append(Cache c, Batch b, Rows kr, Rows vr) {
  constexpr int TPR = D / 8, RPP = 256 / TPR;  // threads per row, rows per pass
  constexpr int MAXB = PASSES * RPP < 128 ? PASSES * RPP : 128;
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t tile[D * MAXB];
  Seq s;
  int within;
  const int head = (int)(blockIdx.x % (unsigned)c.n_kv);
  if (!find_item(b, c.lb, (int)(blockIdx.x / (unsigned)c.n_kv), [&](const Seq& q) { return blocks_touched(q, c.lb); },
                 s, within))
    return;
  const bool is_v = blockIdx.y != 0;
  const int B = 1 << c.lb, j = (max(s.pos0, 0) >> c.lb) + within;
  const int id = block_id(b, s.i, j, c.n_blocks);
  if (id < 0) return;
  const int p0 = j << c.lb;
  const int r0 = max(max(s.pos0, 0) - p0, 0);                 // first new row of the block
  const int r1 = min(min(s.pos0 + s.rows, s.len) - p0, B);    // end of its new rows
  const Rows& src = is_v ? vr : kr;
  const int tr = (int)threadIdx.x / TPR, d0 = (int)threadIdx.x % TPR * 8;
  float f[PASSES][8];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + tr;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[p][i] = 0.f;
    if (r >= r0 && r < r1) {
      load8<SRC32>(src.p, (s.row0 + (long long)(p0 + r - s.pos0)) * src.ts + head * src.hs + d0, f[p]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = fabsf(f[p][i]);
      if (x < INFINITY) amax = fmaxf(amax, x);  // the scale is that of the finite values
    }
  }
  amax = block_max<4>(amax, red);
  float* sp = (is_v ? c.vs : c.ks) + (long long)id * c.n_kv + head;
  int e = scale_exp(amax);
  float ratio = 1.f;  // old scale / new scale
  if (r0 > 0) {
    const float old = *sp;
    const int eo = old > 0.f ? max(min(ilogbf(old), 127), -126) : -126;
    ratio = eo < e ? ldexpf(1.f, eo - e) : 1.f;
    e = max(e, eo);
  }
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *sp = ldexpf(1.f, e);
  const Unscale u = unscale(e);
  uint8_t* dst = (is_v ? c.v : c.k) + ((long long)id * c.n_kv + head) * ((long long)D << c.lb);
  if (!is_v) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int r = p * RPP + tr;
      u32x2* w = reinterpret_cast<u32x2*>(dst + (long long)r * D + d0);
      if (r >= r0 && r < r1) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f[p][i] * u.f * u.g;
        *w = u32x2{encode4(x[0], x[1], x[2], x[3]), encode4(x[4], x[5], x[6], x[7])};
      } else if (r < r0 && ratio < 1.f) {
        const u32x2 o = *w;
        *w = u32x2{rescale4(o.x, ratio), rescale4(o.y, ratio)};
      }
    }
    return;
  }
  // V: the codes turn in LDS to [D][B]; 16 rows of one dimension make a piece
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * RPP + tr;
    if (r >= r0 && r < r1) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = f[p][i] * u.f * u.g;
      const uint32_t w[2] = {encode4(x[0], x[1], x[2], x[3]), encode4(x[4], x[5], x[6], x[7])};
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[(d0 + i) * B + r] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
  __syncthreads();
  const int c0 = ratio < 1.f ? 0 : r0 >> 4, c1 = (r1 + 15) >> 4;  // pieces that change
  const int n = D * (c1 - c0);
  for (int i = (int)threadIdx.x; i < n; i += 256) {
    const int d = i / (c1 - c0), pc = c0 + i % (c1 - c0);
    u32x4* w = reinterpret_cast<u32x4*>(dst + (long long)d * B + pc * 16);
    u32x4 x = *reinterpret_cast<const u32x4*>(tile + d * B + pc * 16);
    if (pc * 16 < r0 || pc * 16 + 16 > r1) {  // some rows of the piece are old, or not written yet
      const u32x4 o = *w;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t os = ratio < 1.f ? rescale4(o[q], ratio) : o[q];
        uint32_t m_new = 0, m_old = 0;
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int r = pc * 16 + 4 * q + z;
          if (r >= r0 && r < r1) m_new |= 0xffu << (8 * z);
          if (r < r0) m_old |= 0xffu << (8 * z);
        }
        x[q] = (x[q] & m_new) | (os & m_old) | (o[q] & ~(m_new | m_old));
      }
    }
    *w = x;
  }
}

// --------------------------------------------------------------- read back
// One workgroup per (block, head, K or V), as the append.  Rows of missing
// blocks, and rows before position 0, are written as zeros.
__device__ __forceinline__ void decode8(u32x2 w, float s, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    f[4 * i] = lo[0] * s, f[4 * i + 1] = lo[1] * s, f[4 * i + 2] = hi[0] * s, f[4 * i + 3] = hi[1] * s;
  }
}

// The blocks of every row of a sequence, from position pos0 (rounded down to
// a block; the rows before position 0 and past the table among them).
__device__ __forceinline__ int blocks_spanned(const Seq& s, int lb) {
  return s.rows > 0 ? ((s.pos0 + s.rows - 1) >> lb) - (s.pos0 >> lb) + 1 : 0;
}

template <int D, bool DST32>
__global__ __launch_bounds__(256) void read_back(Cache c, Batch b, Rows kr, Rows vr) {
  constexpr int TPR = D / 8, RPP = 256 / TPR;
  __shared__ __align__(16) uint8_t tile[D * 128];
  Seq s;
  int within;
  const int head = (int)(blockIdx.x % (unsigned)c.n_kv);
  if (!find_item(b, c.lb, (int)(blockIdx.x / (unsigned)c.n_kv), [&](const Seq& q) { return blocks_spanned(q, c.lb); },
                 s, within))
    return;
  const bool is_v = blockIdx.y != 0;
  const int B = 1 << c.lb, j = (s.pos0 >> c.lb) + within;
  const int id = block_id(b, s.i, j, c.n_blocks);
  const int p0 = j * B, r0 = max(s.pos0 - p0, 0), r1 = min(s.pos0 + s.rows - p0, B);
  const int live = min(max(s.len - p0, 0), B);  // rows of the block that hold positions
  const Rows& dst = is_v ? vr : kr;
  const long long off = ((long long)id * c.n_kv + head) * ((long long)D << c.lb);
  const float sc = id >= 0 ? (is_v ? c.vs : c.ks)[(long long)id * c.n_kv + head] : 0.f;
  if (is_v && id >= 0) {
    for (int i = (int)threadIdx.x; i < D * B / 16; i += 256)
      reinterpret_cast<u32x4*>(tile)[i] = reinterpret_cast<const u32x4*>(c.v + off)[i];
  }
  __syncthreads();
  const int tr = (int)threadIdx.x / TPR, d0 = (int)threadIdx.x % TPR * 8;
  for (int r = r0 + tr; r < r1; r += RPP) {
    u32x2 w = u32x2{0, 0};
    if (id >= 0 && r < live) {
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)tile[(d0 + i) * B + r] << (8 * (i & 3));
      } else {
        w = *reinterpret_cast<const u32x2*>(c.k + off + (long long)r * D + d0);
      }
    }
    float f[8];
    decode8(w, sc, f);
    store8<DST32>(dst.p, (s.row0 + (long long)(p0 + r - s.pos0)) * dst.ts + head * dst.hs + d0, f);
  }
}

// --------------------------------------------------------------- attention
// Query rows of one KV head: row r of a sequence is token r / G, query head
// r % G of the group of G that share the KV head.
struct Attn {
  Cache c;
  Batch b;
  Rows q, out;
  int n_q, group;
  float scale;      // softmax scale * log2(e)
  float* part;      // partials of the splits (null: one split)
  int max_splits, min_tiles;
};

constexpr int ROWS = 16;  // query rows of a row tile (the matrix columns)
constexpr int TILE = 64;  // positions of a step

// Splits of a row tile that sees `tiles` steps of positions: as many as the
// launch has, with at least min_tiles steps in each.
__device__ __forceinline__ int splits_for(int tiles, int max_splits, int min_tiles) {
  return min(max((tiles + min_tiles - 1) / min_tiles, 1), max_splits);
}
// Floats of one row's partial: D outputs, then the maximum and the sum.
template <int D>
__device__ __forceinline__ float* part_at(float* part, long long row, int max_splits, int s) {
  return part + (row * max_splits + s) * (D + 2);
}

// Codes of the value NaN (0x7f, 0xff) in four bytes: 0x80 in each such byte.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int D>
__global__ __launch_bounds__(256) void attn_rows(Attn p) {
  constexpr int KH = D / 64, DT = D / 16;  // 64-dimension halves of K, 16-dimension tiles of V
  __shared__ float lm[4][ROWS], ls[4][ROWS];
  __shared__ float lo[4][ROWS][D + 1];
  const int lb = p.c.lb, G = p.group;
  const int head = (int)(blockIdx.x % (unsigned)p.c.n_kv);
  Seq s;
  int rt;
  if (!find_item(p.b, lb, (int)(blockIdx.x / (unsigned)p.c.n_kv),
                 [&](const Seq& x) { return (int)(((long long)x.rows * G + ROWS - 1) / ROWS); }, s, rt))
    return;
  const int l = (int)(threadIdx.x & 63u), wv = wave_id();
  const int c = l & 15, g = l >> 4;  // this lane's query row; its 16 positions of a step
  const int r0 = rt * ROWS, r = r0 + c;
  const int n_rows = (int)min((long long)s.rows * G - r0, (long long)ROWS);
  const bool mine = c < n_rows;
  const int tok = (mine ? r : r0) / G, hd = head * G + (mine ? r : r0) % G;
  // positions that this row sees: [0, see)
  const int see = mine ? min(max(s.pos0 + tok + 1, 0), s.len) : 0;
  const int see_all = min(max(s.pos0 + r0 / G + 1, 0), s.len);                     // seen by every row
  const int see_any = min(max(s.pos0 + (r0 + n_rows - 1) / G + 1, 0), s.len);  // seen by some row
  const int tiles = (see_any + TILE - 1) / TILE;
  const int ns = splits_for(tiles, p.max_splits, p.min_tiles), sp = (int)blockIdx.y;
  if (sp >= ns) return;
  const int t0 = (int)((long long)tiles * sp / ns), t1 = (int)((long long)tiles * (sp + 1) / ns);

  bf16x8 qv[2 * KH];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(p.q.p) + (s.row0 + tok) * p.q.ts + hd * p.q.hs;
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qv[2 * h + e] = *reinterpret_cast<const bf16x8*>(qp + 64 * h + 16 * g + 8 * e);
  }
  f32x4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, sum = 0.f;
  const int a = c >> 2, bb = c & 3;  // a K load's lane holds position 16a + 4t + bb of the step

  for (int t = t0 + wv; t < t1; t += 4) {
    const int pk = t * TILE + 16 * a, pv = t * TILE + 16 * g;
    int ik = pk < s.len ? block_id(p.b, s.i, pk >> lb, p.c.n_blocks) : -1;
    int iv = pv < s.len ? block_id(p.b, s.i, pv >> lb, p.c.n_blocks) : -1;
    const bool gone = iv < 0;
    ik = max(ik, 0);  // a missing block's place is taken by block 0, masked below
    iv = max(iv, 0);
    const uint8_t* kp = p.c.k + (((long long)ik * p.c.n_kv + head) * D << lb) + (long long)((pk & ((1 << lb) - 1)) + bb) * D + 16 * g;
    const uint8_t* vp = p.c.v + (((long long)iv * p.c.n_kv + head) * D << lb) + ((long long)c << lb) + (pv & ((1 << lb) - 1));
    const float ks = p.c.ks[(long long)ik * p.c.n_kv + head];
    // block 0 may never have been written: its scale must not turn 0 into NaN
    const float vs = gone ? 1.f : p.c.vs[(long long)iv * p.c.n_kv + head];
    u32x4 kw[4][KH], vw[DT];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int h = 0; h < KH; ++h) kw[x][h] = *reinterpret_cast<const u32x4*>(kp + 4 * x * D + 64 * h);
#pragma unroll
    for (int d = 0; d < DT; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + ((long long)(16 * d) << lb));

    f32x4 sc[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      sc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x4 k8 = fp8x8_to_bf16x8_scaled(u32x2{kw[x][h][2 * e], kw[x][h][2 * e + 1]}, ks);
          sc[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k8), qv[2 * h + e], sc[x], 0, 0, 0);
        }
    }
    // scores of positions pv + 4x + i of row c
    const bool masked = (t + 1) * TILE > see_all || __any(gone);
    if (masked) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool vis = !gone && pv + 4 * x + i < see;
          sc[x][i] = vis ? sc[x][i] : -INFINITY;
        }
      // A NaN in V must not reach the rows that do not see it (0 * NaN): it
      // is taken out here, and put into the rows that do see it.
      uint32_t bad = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= nan_bytes(vw[d][i]);
      if (__any(bad)) {
        bf16x8 seen[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i) seen[e][i] = (__bf16)((!gone && pv + 8 * e + i < see) ? 1.f : 0.f);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4 hit = f32x4{0.f, 0.f, 0.f, 0.f};
          u32x4 is;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t n = nan_bytes(vw[d][i]) >> 7;  // 1 in each NaN byte
            is[i] = n * 0x38u;                            // e4m3 of 1
            vw[d][i] &= ~(n * 0xffu);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, fp8x8_to_bf16x8_scaled(u32x2{is[2 * e], is[2 * e + 1]}, 1.f)), seen[e], hit, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = hit[i] > 0.f ? NAN : o[d][i];
        }
      }
    }
    float mt = sc[0][0];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, sc[x][i]);
    mt = max_xor32(max_xor16(mt)) * p.scale;
    const float mn = fmaxf(m, mt), mref = mn == -INFINITY ? 0.f : mn;
    const float al = __builtin_amdgcn_exp2f(m - mref);
    m = mn;
    float pr[16], add = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pr[4 * x + i] = __builtin_amdgcn_exp2f(fmaf(sc[x][i], p.scale, -mref));
        add += pr[4 * x + i];
      }
    sum = sum * al + add;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= al;
    bf16x8 pb[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const bf16x2 w = __builtin_convertvector(f32x2{pr[8 * e + i], pr[8 * e + i + 1]}, bf16x2);
        pb[e][i] = w[0];
        pb[e][i + 1] = w[1];
      }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x4 v8 = fp8x8_to_bf16x8_scaled(u32x2{vw[d][2 * e], vw[d][2 * e + 1]}, vs);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v8), pb[e], o[d], 0, 0, 0);
      }
  }
  sum = sum_xor32(sum_xor16(sum));

  // join the four waves: o[d][i] is dimension 16d + 4g + i of row c
  if (g == 0) lm[wv][c] = m, ls[wv][c] = sum;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[wv][c][16 * d + 4 * g + i] = o[d][i];
  __syncthreads();
  const int row = (int)threadIdx.x / 16, q16 = (int)threadIdx.x % 16;
  if (row >= n_rows) return;
  float mm = lm[0][row];
#pragma unroll
  for (int w = 1; w < 4; ++w) mm = fmaxf(mm, lm[w][row]);
  const float mref = mm == -INFINITY ? 0.f : mm;
  float wt[4], tot = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    wt[w] = __builtin_amdgcn_exp2f(lm[w][row] - mref);
    tot += wt[w] * ls[w][row];
  }
  const int tk = (r0 + row) / G, oh = head * G + (r0 + row) % G;
  const float inv = ns == 1 ? (tot > 0.f || tot != tot ? 1.f / tot : 0.f) : 1.f;
  float y[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int d = q16 * (D / 16) + i;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v += wt[w] * lo[w][row][d];
    y[i] = v * inv;
  }
  if (ns == 1) {
    uint16_t* op = static_cast<uint16_t*>(p.out.p) + (s.row0 + tk) * p.out.ts + oh * p.out.hs + q16 * (D / 16);
#pragma unroll
    for (int i = 0; i < D / 16; i += 2)
      *reinterpret_cast<uint32_t*>(op + i) = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{y[i], y[i + 1]}, bf16x2));
  } else {
    float* pp = part_at<D>(p.part, (long long)(s.row0 + tk) * p.n_q + oh, p.max_splits, sp);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) pp[q16 * (D / 16) + i] = y[i];
    if (q16 == 0) pp[D] = mm, pp[D + 1] = tot;
  }
}

// Joins the splits of every row that has more than one, in the splits' order.
template <int D>
__global__ __launch_bounds__(256) void attn_join(Attn p) {
  const int lb = p.c.lb, G = p.group;
  const int head = (int)(blockIdx.x % (unsigned)p.c.n_kv);
  Seq s;
  int rt;
  if (!find_item(p.b, lb, (int)(blockIdx.x / (unsigned)p.c.n_kv),
                 [&](const Seq& x) { return (int)(((long long)x.rows * G + ROWS - 1) / ROWS); }, s, rt))
    return;
  const int r0 = rt * ROWS, n_rows = (int)min((long long)s.rows * G - r0, (long long)ROWS);
  const int see_any = min(max(s.pos0 + (r0 + n_rows - 1) / G + 1, 0), s.len);
  const int ns = splits_for((see_any + TILE - 1) / TILE, p.max_splits, p.min_tiles);
  if (ns == 1) return;
  for (int i = (int)threadIdx.x; i < n_rows * D; i += 256) {
    const int row = i / D, d = i % D, tk = (r0 + row) / G, oh = head * G + (r0 + row) % G;
    const float* pp = part_at<D>(p.part, (long long)(s.row0 + tk) * p.n_q + oh, p.max_splits, 0);
    float mm = -INFINITY;
    for (int z = 0; z < ns; ++z) mm = fmaxf(mm, pp[z * (D + 2) + D]);
    const float mref = mm == -INFINITY ? 0.f : mm;
    float v = 0.f, tot = 0.f;
    for (int z = 0; z < ns; ++z) {
      const float w = __builtin_amdgcn_exp2f(pp[z * (D + 2) + D] - mref);
      v += w * pp[z * (D + 2) + d];
      tot += w * pp[z * (D + 2) + D + 1];
    }
    const float y = tot > 0.f || tot != tot ? v / tot : 0.f;
    static_cast<uint16_t*>(p.out.p)[(s.row0 + tk) * p.out.ts + oh * p.out.hs + d] =
        __builtin_bit_cast(uint16_t, (__bf16)y);
  }
}

}  // namespace kv8
}  // namespace mk
