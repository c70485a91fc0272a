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

template <int V>
struct Int {
  static constexpr int value = V;
};

// Sum over the lanes up to and with this one (DPP: no step through LDS).
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 -> 1, 2 -> 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // rows 0, 1 -> 2, 3
  return x;
}

// Work items are dealt to the sequences in order, count(seq) each; finds the
// sequence of item `it` and the item's number within it.  A wave looks at 64
// sequences at a time (the whole wave must call it), each lane at one, so a
// workgroup waits for one round of loads.  False past the last.
template <class Count>
__device__ __forceinline__ bool find_item(const Batch& b, int lb, int it, Count count, Seq& s, int& within) {
  const int l = (int)(threadIdx.x & (kWave - 1u));
  int before = 0;
  for (int base = 0; base < b.n_seq; base += kWave) {
    Seq q{};
    int c = 0;
    if (base + l < b.n_seq) {
      q = seq_at(b, base + l, lb);
      c = count(q);
    }
    const int sum = wave_prefix(c);
    const unsigned long long hit = __ballot(before + sum > it);
    if (hit) {
      const int f = __builtin_amdgcn_readfirstlane(__ffsll((long long)hit) - 1);
      s.i = base + f;
      s.row0 = __builtin_amdgcn_readlane(q.row0, f);
      s.rows = __builtin_amdgcn_readlane(q.rows, f);
      s.pos0 = __builtin_amdgcn_readlane(q.pos0, f);
      s.len = __builtin_amdgcn_readlane(q.len, f);
      within = it - before - (__builtin_amdgcn_readlane(sum, f) - __builtin_amdgcn_readlane(c, f));
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, kWave - 1);
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
// would be off by 2^-24 of an angle of up to 1e5 radians; fp64's roundings are
// off by 2^-52); the sine and cosine of the fraction are fp32.  Every head
// forms its own.  8,192 tokens of 24 heads of 128, fp32 to bf16 (151 MB), take
// 28 us, 5.4 TB/s; bf16 in place (101 MB) 22.5, 4.5 TB/s, and of 64 (50 MB)
// 15.7, 3.2 TB/s, where the arithmetic is no longer behind the loads; 16 tokens
// 2.7 us in a graph, where an empty launch takes as long.
template <int D, bool SRC32, bool DST32>
__global__ __launch_bounds__(256) void norm_rope(Rows q, Rows k, const uint16_t* __restrict__ qg,
                                                 const uint16_t* __restrict__ kg, const float* __restrict__ freq,
                                                 const int* __restrict__ pos, Rows qo, Rows ko, int n_tokens, int n_q,
                                                 int n_kv, float eps) {
  constexpr int LPH = D / 16, HPW = kWave / LPH;  // lanes per head, heads per wave
  const int l = (int)(threadIdx.x & 63u), j = l % LPH;
  const int heads = n_q + n_kv, passes = (heads + HPW - 1) / HPW;
  const unsigned it = blockIdx.x * 4 + threadIdx.x / 64;  // below 2^26
  const int t = (int)(it / (unsigned)passes), h = (int)(it % (unsigned)passes) * HPW + l / LPH;
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
// (448 = 1.75 * 2^8), but at most 2^119: beyond, codes times the scale would
// pass fp32's and bf16's largest values, and an infinite value reaches rows
// that do not see it (0 * inf).  Zero rows give 2^-126, so that a block that
// starts with them takes the scale of the rows that follow.
constexpr float kTop = 0x1.cp127f;  // 448 * 2^119
__device__ __forceinline__ int scale_exp(float amax) {
  if (!(amax > 0.f)) return -126;
  int e = ilogbf(amax) - 8;
  if (amax > ldexpf(448.f, e)) ++e;
  return min(max(e, -126), 119);
}

// Codes of four values that were divided by the scale: nearest, ties to even.
// The values are within 448, or saturate()d.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Infinities, and what is beyond 448 s of the largest scale, to +-448; NaN stays.
__device__ __forceinline__ float saturate(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }

// Four codes re-rounded after multiplying by a power of two of at most one.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return encode4(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}

// A block's rows are dealt to threads in pieces of 4 rows x W dimensions (8;
// 4 where rows are written in fp32): in K a piece is W consecutive bytes of 4
// rows, in V 4 consecutive bytes of W dimensions, so neither layout needs a
// transposition through LDS, and in the rows it is 16 consecutive bytes (32
// of fp32 input).  A wave holds 32 rows x 8W dimensions (16 rows x 16W of the
// smallest block), where 64 consecutive bytes of K, 32 of V and 128 of a row
// are touched at once.
struct Piece {
  int row, dim;
};
template <int D, int W>
__device__ __forceinline__ Piece piece_at(int u, int lb) {
  // u: row quad (3 bits, 2 for blocks of 16), dimension group (the rest of 6 bits, if there are so many), then the rest
  constexpr int gb = (D == 64 ? 6 : 7) - (W == 8 ? 3 : 2);  // log2 of the groups of W dimensions
  const int qb = min(lb - 2, 3), ob = min(6 - qb, gb);
  const int hi = u >> (qb + ob), qh = lb - 2 - qb;  // row quads beyond the first 8
  return Piece{((u & ((1 << qb) - 1)) | (hi & ((1 << qh) - 1)) << qb) * 4, ((u >> qb & ((1 << ob) - 1)) | hi >> qh << ob) * W};
}

// Eight elements of a row as they were loaded (once, so past the caches).
template <bool F32>
struct Raw8 {
  u32x4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, long long e) {
    const u32x4* q = F32 ? reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + e)
                         : reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = __builtin_nontemporal_load(q + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (F32) return __uint_as_float(w[e >> 2][e & 3]);
    else return e & 1 ? bf16_hi(w[0][e >> 1]) : bf16_lo(w[0][e >> 1]);
  }
  // Largest magnitude so far, as bits (whose order is that of the values,
  // infinities above and NaN above those): of one fp32, or of two bf16 side
  // by side.
  __device__ __forceinline__ void top(uint32_t& m) const {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (F32) m = max(m, w[i][j] & 0x7fffffffu);
        else
          m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                     __builtin_bit_cast(u16x2, w[i][j] & 0x7fff7fffu)));
      }
  }
  static __device__ __forceinline__ float top_value(uint32_t m) {
    return __uint_as_float(F32 ? m : max(m & 0xffff0000u, m << 16));
  }
};

// One team of T threads per block that rows go to and head, K and V both; a
// workgroup holds 256 / T heads.  The rows stay in registers as they were
// loaded between the maximum and the rounding, so the input is read once (66
// registers from bf16; expanded to fp32 it took 104, and 35 us where this takes
// 24: 16,499 rows of 8 heads of 128 in ragged prompts, 101 MB, 4.2 TB/s; from
// fp32 41 us, 169 MB, 4.1 TB/s).  One row to each of 16 sequences takes 6 us: three loads in a row (lengths, table,
// rows) and the launch.
template <int D, int T, int PASSES, bool SRC32>
__global__ __launch_bounds__(256) void append(Cache c, Batch b, Rows kr, Rows vr) {
  constexpr int HEADS = 256 / T;
  __shared__ float red[4][2];
  Seq s;
  int within;
  const unsigned sets = (unsigned)((c.n_kv + HEADS - 1) / HEADS);
  if (!find_item(b, c.lb, (int)(blockIdx.x / sets), [&](const Seq& q) { return blocks_touched(q, c.lb); }, s, within)) return;
  const int tid = (int)threadIdx.x, head = (int)(blockIdx.x % sets) * HEADS + tid / T;
  const int B = 1 << c.lb, j = (max(s.pos0, 0) >> c.lb) + within;
  const int id = block_id(b, s.i, j, c.n_blocks);
  if (id < 0) return;
  const bool on = head < c.n_kv;
  const int p0 = j << c.lb;
  const int r0 = max(max(s.pos0, 0) - p0, 0);               // first new row of the block
  const int r1 = min(min(s.pos0 + s.rows, s.len) - p0, B);  // end of its new rows
  const long long at = (long long)id * c.n_kv + head;
  float old_k = 0.f, old_v = 0.f;
  if (r0 > 0 && on) old_k = c.ks[at], old_v = c.vs[at];
  Raw8<SRC32> kr8[PASSES][4], vr8[PASSES][4];
  uint32_t vold[PASSES][8];  // V's dwords, where a piece has rows that stay
  uint32_t ktop = 0, vtop = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const Piece pc = piece_at<D, 8>(tid % T + p * T, c.lb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = pc.row + i;
      const long long row = s.row0 + (long long)(p0 + r - s.pos0);
      kr8[p][i].zero();
      vr8[p][i].zero();
      if (on && r >= r0 && r < r1) {
        kr8[p][i].load(kr.p, row * kr.ts + head * kr.hs + pc.dim);
        vr8[p][i].load(vr.p, row * vr.ts + head * vr.hs + pc.dim);
      }
    }
    if (on && pc.row < r1 && (pc.row < r0 || pc.row + 4 > r1)) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vold[p][e] = *reinterpret_cast<const uint32_t*>(c.v + ((at * D + pc.dim + e) << c.lb) + pc.row);
    }
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kr8[p][i].top(ktop);
      vr8[p][i].top(vtop);
    }
  float kmax = Raw8<SRC32>::top_value(ktop), vmax = Raw8<SRC32>::top_value(vtop);
  const bool odd = __any(!(kmax <= kTop) || !(vmax <= kTop));  // some value is no finite number, or too large for any scale
  if (__builtin_expect(odd, 0)) {                              // the scale is that of the finite values
    kmax = vmax = 0.f;
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = fabsf(kr8[p][i].get(e)), y = fabsf(vr8[p][i].get(e));
          kmax = fmaxf(kmax, x < INFINITY ? x : 0.f);
          vmax = fmaxf(vmax, y < INFINITY ? y : 0.f);
        }
  }
  kmax = max_xor16(group_max<16>(kmax));
  vmax = max_xor16(group_max<16>(vmax));
  if constexpr (T >= 64) {
    kmax = max_xor32(kmax);
    vmax = max_xor32(vmax);
  }
  if constexpr (T > 64) {
    if (tid % 64 == 0) red[tid / 64][0] = kmax, red[tid / 64][1] = vmax;
    __syncthreads();
    const int w = tid / T * (T / 64);
#pragma unroll
    for (int i = 0; i < T / 64; ++i) kmax = fmaxf(kmax, red[w + i][0]), vmax = fmaxf(vmax, red[w + i][1]);
  }
  if (!on) return;
  // the block's scale, and old scale / new scale
  const auto settle = [&](float amax, float old, float& ratio) {
    int e = scale_exp(amax);
    ratio = 1.f;
    if (r0 > 0) {
      const int eo = old > 0.f ? max(min(ilogbf(old), 127), -126) : -126;
      if (eo < e) ratio = ldexpf(1.f, eo - e);
      e = max(e, eo);
    }
    return e;
  };
  float kratio, vratio;
  const int ke = settle(kmax, old_k, kratio), ve = settle(vmax, old_v, vratio);
  if (tid % T == 0) {  // the team's old scales were read before its maxima met
    c.ks[at] = ldexpf(1.f, ke);
    c.vs[at] = ldexpf(1.f, ve);
  }
  const float ku = ldexpf(1.f, -ke), vu = ldexpf(1.f, -ve);
  uint8_t *kd = c.k + (at * D << c.lb), *vd = c.v + (at * D << c.lb);
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const Piece pc = piece_at<D, 8>(tid % T + p * T, c.lb);
    if (pc.row >= r1) continue;
    const auto code4 = [&](float x, float y, float z, float w) {
      if (__builtin_expect(odd, 0)) x = saturate(x), y = saturate(y), z = saturate(z), w = saturate(w);
      return encode4(x, y, z, w);
    };
    uint32_t keep = 0, older = 0;  // bytes of V's dwords that stay as they are; those of older rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = pc.row + i;
      u32x2* w = reinterpret_cast<u32x2*>(kd + (long long)r * D + pc.dim);
      if (r >= r0 && r < r1) {
        const Raw8<SRC32>& x = kr8[p][i];
        *w = u32x2{code4(x.get(0) * ku, x.get(1) * ku, x.get(2) * ku, x.get(3) * ku),
                   code4(x.get(4) * ku, x.get(5) * ku, x.get(6) * ku, x.get(7) * ku)};
      } else {
        keep |= 0xffu << (8 * i);
        if (r < r0) {
          older |= 0xffu << (8 * i);
          if (kratio < 1.f) *w = u32x2{rescale4(w->x, kratio), rescale4(w->y, kratio)};
        }
      }
    }
    if (keep == 0xffffffffu && !(older && vratio < 1.f)) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t x = code4(vr8[p][0].get(e) * vu, vr8[p][1].get(e) * vu, vr8[p][2].get(e) * vu, vr8[p][3].get(e) * vu);
      if (keep) {
        const uint32_t o = vold[p][e], os = vratio < 1.f ? rescale4(o, vratio) : o;
        x = (x & ~keep) | (os & older) | (o & keep & ~older);
      }
      *reinterpret_cast<uint32_t*>(vd + ((long long)(pc.dim + e) << c.lb) + pc.row) = x;
    }
  }
}

// --------------------------------------------------------------- read back
// Rows of missing blocks, and rows before position 0, are written as zeros.
__device__ __forceinline__ void decode4(uint32_t w, float s, float* f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = lo[0] * s, f[1] = lo[1] * s, f[2] = hi[0] * s, f[3] = hi[1] * s;
}
// 16 bytes of a row: 8 bf16 or 4 fp32.  Past the caches: nothing here reads
// them again, and as ordinary stores they pushed out codes that were still to
// be read (16 contexts of 512 to 4,096 into fp32, 377 MB: 94 us, now 66,
// 5.7 TB/s).
template <bool F32>
__device__ __forceinline__ void put16(void* p, long long e, const float* f) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F32) w[i] = __float_as_uint(f[i]);
    else w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{f[2 * i], f[2 * i + 1]}, bf16x2));
  }
  u32x4* q = F32 ? reinterpret_cast<u32x4*>(static_cast<float*>(p) + e) : reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + e);
  __builtin_nontemporal_store(w, q);
}

// The blocks of every row of a sequence, from position pos0 (rounded down to
// a block; the rows before position 0 and past the table among them).
__device__ __forceinline__ int blocks_spanned(const Seq& s, int lb) {
  return s.rows > 0 ? ((s.pos0 + s.rows - 1) >> lb) - (s.pos0 >> lb) + 1 : 0;
}

// Bytes 0..3 of the result: byte i of a, b, c, d.
__device__ __forceinline__ uint32_t gather4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int i) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, (uint32_t)i | (uint32_t)(4 + i) << 8);
  const uint32_t hi = __builtin_amdgcn_perm(d, c, (uint32_t)i | (uint32_t)(4 + i) << 8);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// A workgroup takes `heads` heads of one block; a thread a piece at a time.
// Bound by the bytes: the same rows back as bf16 20 us (101 MB, 5.1 TB/s).
template <int D, bool DST32>
__global__ __launch_bounds__(256) void read_back(Cache c, Batch b, Rows kr, Rows vr, int heads) {
  Seq s;
  int within;
  const unsigned sets = (unsigned)((c.n_kv + heads - 1) / heads);
  if (!find_item(b, c.lb, (int)(blockIdx.x / sets), [&](const Seq& q) { return blocks_spanned(q, c.lb); }, s, within)) return;
  const int B = 1 << c.lb, j = (s.pos0 >> c.lb) + within, h0 = (int)(blockIdx.x % sets) * heads;
  const int id = block_id(b, s.i, j, c.n_blocks);
  const int p0 = j * B, r0 = max(s.pos0 - p0, 0), r1 = min(s.pos0 + s.rows - p0, B);
  const int live = id >= 0 ? min(max(s.len - p0, 0), B) : 0;  // rows of the block that hold positions
  constexpr int W = DST32 ? 4 : 8, ND = W / 4;
  const int lu = c.lb - 2 + (D == 64 ? 6 : 7) - (W == 8 ? 3 : 2);  // log2 of a head's pieces
  const int n = min(heads, c.n_kv - h0) << lu;
  for (int u = (int)threadIdx.x; u < n; u += 256) {
    const int head = h0 + (u >> lu);
    const Piece pc = piece_at<D, W>(u & ((1 << lu) - 1), c.lb);
    if (pc.row + 4 <= r0 || pc.row >= r1) continue;
    uint32_t kw[4][ND], vw[W];
    float ks = 0.f, vs = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < ND; ++j) kw[i][j] = 0;
#pragma unroll
    for (int e = 0; e < W; ++e) vw[e] = 0;
    if (pc.row < live) {  // the whole piece lies in the block; rows past `live` are dropped below
      const long long at = (long long)id * c.n_kv + head;
      const uint8_t *kp = c.k + (at * D << c.lb) + pc.row * D + pc.dim, *vp = c.v + (at * D << c.lb) + (pc.dim << c.lb) + pc.row;
      ks = c.ks[at], vs = c.vs[at];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (W == 8) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(kp + i * D);
          kw[i][0] = x.x, kw[i][ND - 1] = x.y;
        } else {
          kw[i][0] = *reinterpret_cast<const uint32_t*>(kp + i * D);
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e) vw[e] = *reinterpret_cast<const uint32_t*>(vp + (e << c.lb));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = pc.row + i;
      if (r < r0 || r >= r1) continue;
      const bool is = r < live;
      const long long row = s.row0 + (long long)(p0 + r - s.pos0);
      float f[W];
#pragma unroll
      for (int j = 0; j < ND; ++j) decode4(is ? kw[i][j] : 0u, is ? ks : 0.f, f + 4 * j);
      put16<DST32>(kr.p, row * kr.ts + head * kr.hs + pc.dim, f);
#pragma unroll
      for (int j = 0; j < ND; ++j)
        decode4(is ? gather4(vw[4 * j], vw[4 * j + 1], vw[4 * j + 2], vw[4 * j + 3], i) : 0u, is ? vs : 0.f, f + 4 * j);
      put16<DST32>(vr.p, row * vr.ts + head * vr.hs + pc.dim, f);
    }
  }
}

// --------------------------------------------------------------- attention
// Query rows of one KV head: row r of a sequence is token r / G, query head
// r % G of the group of G that share the KV head.
// How the work of one kernel is dealt out: row tiles of 2^lr rows, and where
// contexts are split the steps of positions of all row tiles in about
// `target` items per KV head, of at least `least` steps each; target 0 for no
// splits.  Partials: outputs [slot][head][row][D] and maxima and sums
// [slot][head][row].
struct Deal {
  int lr, target, least, items;
  float* part;
  float2* ml;
};

enum Kind : int { FEW = 0, MANY = 1 };  // attn_rows, attn_tile

struct Attn {
  Cache c;
  Batch b;
  Rows q, out;
  int n_q, group;
  float scale;  // softmax scale * log2(e)
  int few;      // sequences of up to so many query rows are attn_rows's, the others attn_tile's
  Deal d[2];
};

// What a score is beyond scale * q . k, and which positions a row sees beyond
// the causal ones: s = cap * tanh(scale q.k / cap) - slope[head] |p - j| for
// the row at position p and position j, seen if max(first[row], p + 1 -
// window) <= j < max(p + 1, prefix[sequence]).
struct Scores {
  const float* slopes;  // [n_q], or null
  const int* first;     // [n_tokens], or null
  const int* prefix;    // [n_seq], or null
  int window;           // 0: none
  float cap, cap_in;    // cap * log2(e) (0: none), scale / cap
  float c[4];           // cap * log2(e) times the coefficients of Q of score()
};
// The attention with such scores, or with each row's log-sum-exp: the same
// kernels, compiled once more.  Scores are formed less the row's reference, so
// what is not asked for costs a branch a step, a cap seven operations for each
// score (where some pass half of it six, two of them slow), slopes three, the
// log-sum-exp one.  1,024 tokens of 16 / 8 heads of 128 at 16,384 positions: causal 167
// us, with scores 160, capped 196, with slopes 176; four prompts of 2,048 tokens, heads
// of 64, 66, 73, 101 (where most steps pass half the cap 15 % more), 87.  (Of biased
// scores less the reference from the start near ones were rounded beside far ones'
// biases, which log-sum-exps showed; 3 to 5 % less time.)  Steps that a row tile sees
// none of are not walked: a window of 4,096 at 32,768 positions takes 12.5 us, the
// whole 18.  The 128-row tiles without log-sum-exps leave three registers of head_dim
// 128 in scratch memory, with few rows beside them two of 64 (12 to 16 bytes a lane).
struct AttnScored : Attn {
  Scores x;
};
struct AttnLse : AttnScored {
  float* lse;    // [n_tokens][n_q]
  float* ex[2];  // with splits, next to Deal::ml: sums of the weights as they were before their rounding
};
template <class P>
struct Has {
  static constexpr bool scores = __is_base_of(AttnScored, P), lse = __is_base_of(AttnLse, P);
};

constexpr int ROWS = 16;        // query rows of attn_rows's tile (the matrix columns)
constexpr int TILE_ROWS = 128;  // and of attn_tile's
constexpr int TILE = 64;        // positions of a step

// Row tile rt of a sequence: its rows, and the positions [from, any) that some
// row of it sees, [shut, all) that every row sees.
struct RowTile {
  int n_rows, from, shut, any, all;
};
__device__ __forceinline__ RowTile row_tile(const Seq& s, int G, int rt, int rows) {
  const int r0 = rt * rows;  // rows times G are at most 2^30
  RowTile t;
  t.from = t.shut = 0;
  t.n_rows = min(s.rows * G - r0, rows);
  t.all = min(max(s.pos0 + r0 / G + 1, 0), s.len);
  t.any = min(max(s.pos0 + (r0 + t.n_rows - 1) / G + 1, 0), s.len);
  return t;
}
__device__ __forceinline__ int row_tiles(const Seq& s, int G, int lr) {
  return (s.rows * G + (1 << lr) - 1) >> lr;
}

// Largest over the wave.
__device__ __forceinline__ int wave_imax(int v) {
  const auto sel = [](int x, auto ctrl) { return __builtin_amdgcn_update_dpp(0x80000000, x, decltype(ctrl)::value, 0xf, 0xf, false); };
  v = max(v, sel(v, Int<DPP_XOR1>{}));
  v = max(v, sel(v, Int<DPP_XOR2>{}));
  v = max(v, sel(v, Int<DPP_HALF_MIRROR>{}));
  v = max(v, sel(v, Int<DPP_MIRROR>{}));
  auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  v = max((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane(max((int)r[0], (int)r[1]));
}
__device__ __forceinline__ int wave_imin(int v) { return ~wave_imax(~v); }

// Positions [lo, hi) that a row sees; of none both are 0.
struct Sight {
  int lo, hi;
};
__device__ __forceinline__ Sight sight(const Batch& b, const Scores& x, const Seq& s, int tok) {
  const int p = s.pos0 + tok;
  int lo = 0, hi = p + 1;
  if (x.window) lo = (int)max((long long)p + 1 - x.window, 0ll);
  if (x.first) lo = max(lo, x.first[s.row0 + tok]);
  if (x.prefix && p >= 0) hi = max(hi, x.prefix[s.i]);
  hi = min(max(hi, 0), s.len);
  return lo < hi ? Sight{lo, hi} : Sight{0, 0};
}
// The bounds of a row tile from its rows' (each in some lane of the wave).
struct Bounds {
  int from = 0x7fffffff, shut = 0, any = 0, all = 0x7fffffff;
  __device__ __forceinline__ void add(const Sight& v) {
    if (v.hi) from = min(from, v.lo);
    shut = max(shut, v.lo);
    any = max(any, v.hi);
    all = min(all, v.hi);
  }
  __device__ __forceinline__ void join() {
    any = wave_imax(any);
    from = min(wave_imin(from), any);
    shut = wave_imax(shut);
    all = wave_imin(all);
  }
};

// A slope to base 2.  Beyond +-2^94 it counts as that (NaN stays): products with
// distances of up to 2^31 are then finite, and one position further away leaves no
// weight long before.
__device__ __forceinline__ float slope_of(float s) {
  return (s > 0x1p94f ? 0x1p94f : s < -0x1p94f ? -0x1p94f : s) * 1.4426950408889634f;
}

// Scores of one row to base 2 from q . k, with `add` added, in place: N of them,
// at(i) is the position of the i-th less that of the row.  A capped one is cap *
// tanh(y).  Where the wave's are all at most half the cap, tanh(y) = y (1 + y^2 Q(y^2))
// with Q interpolated at Chebyshev's nodes to 2^-24: off by 8 * 2^-24 of itself at
// most.  Else (e^2y - 1) / (e^2y + 1), which e^2y near 1 puts off by 2 * 2^-24 of the
// cap, beside some score that is not small against it.  (1 - 2 / (e^2y + 1) for all
// scores takes 2 to 5 % less, but made log-sum-exps of small ones up to 60 times less
// exact than fp32 has them.)
template <int N, class At>
__device__ __forceinline__ void score(const Scores& x, float scale, float slope, float add, float* s, At at) {
  if (!x.cap) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fmaf(s[i], scale, add);
    asm volatile("");  // branches that stay branches: 64 scores of both kinds at once take registers that are not there
  } else {
    asm volatile("");
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] *= x.cap_in;
      most = fmaxf(most, fabsf(s[i]));
    }
    if (!__any(most > 0.5f)) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float w = s[i] * s[i], q = fmaf(fmaf(fmaf(w, x.c[3], x.c[2]), w, x.c[1]), w, x.c[0]);
        s[i] = fmaf(s[i], fmaf(w, q, x.cap), add);
      }
    } else {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // (e^2y stays finite, and a NaN one)
        const float t = __builtin_amdgcn_exp2f(s[i] > 40.f ? 115.f : s[i] * 2.8853900817779268f);
        s[i] = fmaf((t - 1.f) * x.cap, __builtin_amdgcn_rcpf(t + 1.f), add);
      }
    }
  }
  if (x.slopes) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fmaf(-slope, fabsf((float)at(i)), s[i]);
  }
}

// Most splits of one row tile (attn_join gives each a thread).
constexpr int kMaxSplits = 256;

// A row tile and one of the splits of its positions.
struct Item {
  Seq s;
  int rt, split, ns;  // row tile, split, splits of this sequence's row tiles
  int slot;           // of the tile's first partial, if ns > 1
  int kind;
  // first step of split i, of the row tile's `steps`
  __device__ __forceinline__ int step(int i, int steps) const {
    return ns == 1 ? i * steps : steps / ns * i + min(i, steps % ns);
  }
};

// Steps of a sequence's longest row tile.
__device__ __forceinline__ int most_steps(const Attn&, const Deal&, const Seq& s) {
  return (min(max(s.pos0 + s.rows, 0), s.len) + TILE - 1) / TILE;
}
// With a window those that it lets a row tile see, and one more where it lies
// across steps; documents are not known here.
__device__ __forceinline__ int most_steps(const AttnScored& p, const Deal& d, const Seq& s) {
  if (s.rows <= 0) return 0;
  int hi = max(s.pos0 + s.rows, 0);
  const int prefix = p.x.prefix ? p.x.prefix[s.i] : 0;
  hi = min(max(hi, prefix), s.len);
  int n = (hi + TILE - 1) / TILE;
  if (p.x.window && prefix <= max(s.pos0, 0)) n = (int)min((long long)n, ((long long)p.x.window + (1 << d.lr) / p.group + 2 * TILE) / TILE);
  return n;
}

__device__ __forceinline__ int kind_of(const Attn& p, const Seq& s) { return (long long)s.rows * p.group > p.few; }

// Lane l's sequence of the 64 from `base` on, no rows past the last.
__device__ __forceinline__ Seq lane_seq(const Attn& p, int base) {
  const int i = base + (int)(threadIdx.x & (kWave - 1u));
  return i < p.b.n_seq ? seq_at(p.b, i, p.c.lb) : Seq{};
}

// Steps of an item: the target-th part of all steps of the kernel's row tiles.
// `first` holds the first 64 sequences.
template <class P>
__device__ __forceinline__ int steps_per_item(const P& p, int kind, const Seq& first) {
  const Deal& d = p.d[kind];
  if (!d.target) return 0x7fffffff;
  long long total = 0;
  for (int base = 0; base < p.b.n_seq; base += kWave) {
    const Seq q = base ? lane_seq(p, base) : first;
    const long long w = kind_of(p, q) == kind ? (long long)row_tiles(q, p.group, d.lr) * most_steps(p, d, q) : 0;
    // 64 lanes' sum in two halves that stay inside 32 bits
    const int lo = wave_prefix((int)(w & 0xffffff)), hi = wave_prefix((int)min(w >> 24, 0x1ffffffll));
    total += ((long long)__builtin_amdgcn_readlane(hi, 63) << 24) + __builtin_amdgcn_readlane(lo, 63);
  }
  // (a division of 64 bits takes longer than all the rest)
  const long long per = total < 0x7fffffff ? (int)total / d.target + ((int)total % d.target != 0) : (total + d.target - 1) / d.target;
  return (int)min(max(per, (long long)d.least), 0x7fffffffll);
}

// Where sequences are of unlike length, equal splits of each would leave most
// of the chip waiting for the longest.  Every workgroup therefore adds up the
// steps of all sequences (their lengths are on the device alone), takes the
// `target`-th part of that as the steps of an item, and deals the items out:
// a sequence of k row tiles and n steps gets k * ceil(n / part) of them.
// There are at most target + (row tiles) items, and 2 * target partials: a
// sequence that is split at all has more than one part.
// Finds item `it` of a kernel, or with kind -1 the item that holds token `it`
// of all tokens of kernels that split (r.rt is then the token's number within
// its sequence).
template <int KIND, class P>
__device__ __forceinline__ bool find_split(const P& p, int it, Item& r) {
  const int G = p.group;
  const Seq first = lane_seq(p, 0);
  const int per0 = KIND != MANY ? steps_per_item(p, FEW, first) : 0, per1 = KIND != FEW ? steps_per_item(p, MANY, first) : 0;
  int before = 0, slots0 = 0, slots1 = 0;
  for (int base = 0; base < p.b.n_seq; base += kWave) {
    const Seq q = base ? lane_seq(p, base) : first;
    const int kind = kind_of(p, q);
    int c = 0, s0 = 0, s1 = 0, ns = 1;
    if (KIND < 0 ? (kind ? p.d[1].target : p.d[0].target) != 0 : kind == KIND) {
      const int per = kind ? per1 : per0;
      const int rt = row_tiles(q, G, kind ? p.d[1].lr : p.d[0].lr), n = most_steps(p, kind ? p.d[1] : p.d[0], q);
      if (p.d[0].target | p.d[1].target) ns = min(max(n / per + (n % per != 0), 1), kMaxSplits);
      const int sl = ns > 1 ? rt * ns : 0;
      s0 = kind ? 0 : sl;
      s1 = kind ? sl : 0;
      c = KIND < 0 ? q.rows : rt * ns;
    }
    const int sum = wave_prefix(c), sum0 = KIND != MANY ? wave_prefix(s0) : 0, sum1 = KIND != FEW ? wave_prefix(s1) : 0;
    const unsigned long long hit = __ballot(before + sum > it);
    if (hit) {
      const int f = __builtin_amdgcn_readfirstlane(__ffsll((long long)hit) - 1);
      r.s.i = base + f;
      r.s.row0 = __builtin_amdgcn_readlane(q.row0, f);
      r.s.rows = __builtin_amdgcn_readlane(q.rows, f);
      r.s.pos0 = __builtin_amdgcn_readlane(q.pos0, f);
      r.s.len = __builtin_amdgcn_readlane(q.len, f);
      r.ns = __builtin_amdgcn_readlane(ns, f);
      r.kind = __builtin_amdgcn_readlane(kind, f);
      const int within = it - before - (__builtin_amdgcn_readlane(sum, f) - __builtin_amdgcn_readlane(c, f));
      r.slot = r.kind ? slots1 + __builtin_amdgcn_readlane(sum1 - s1, f) : slots0 + __builtin_amdgcn_readlane(sum0 - s0, f);
      if (KIND < 0) {
        r.rt = within;
        r.split = 0;
      } else {
        r.rt = r.ns == 1 ? within : within / r.ns;
        r.split = within - r.rt * r.ns;
        r.slot += r.rt * r.ns;
      }
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, kWave - 1);
    slots0 += __builtin_amdgcn_readlane(sum0, kWave - 1);
    slots1 += __builtin_amdgcn_readlane(sum1, kWave - 1);
  }
  return false;
}

template <bool V>
struct Bool {
  static constexpr bool value = V;
};

// Weights are exp2(score - reference), where the reference is a row's maximum
// so far, or up to 2^RISE less: sums take a new reference (a product for each
// output held) only where the maximum has risen by more.  Weights of up to 2^8
// lose nothing in bf16 and fp32, and a rise of some maximum of a wave's rows is
// the rule for the first hundred steps.
//
// The weights are rounded to bf16 for the product with V, and what they are
// divided by is the sum of the rounded ones: each is off by up to 2^-8 of
// itself, and against an exact sum a row that one key decides would be off by
// as much as a whole (with the running maximum as the reference its weight is
// 1, with this one any number).  Left is at most 2^-8 sum_j p_j |v_j - out|,
// beside the output's own rounding by up to 2^-8 |out|.  In two bf16 parts,
// with a second product for the lower, outputs are those of fp32 weights, but
// take, us: one token of 16 sequences of 512 to 4,096, head_dim 64, 14.6
// where this takes 13.2; ragged prompts of 33 to 2,048, 71 / 55; 1,024 tokens
// at the end of 32,768 positions, head_dim 128, 417 / 308 (root mean square
// error over that of the values, bf16 outputs: 0.0017 / 0.0020, 0.0017 /
// 0.0019, 0.0017 / 0.0021).  With scores, too: capped decode of 16 sequences of 512 to
// 4,096 19.4 / 17.6, 4,096 tokens in documents 40 / 34.5, 1,024 capped ones at 16,384
// 270 / 213.
constexpr float RISE = 8.f;

// Codes of the value NaN (0x7f, 0xff) in four bytes: 0x80 in each such byte.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t lo, uint32_t hi, float s) {
  return __builtin_bit_cast(bf16x8, fp8x8_to_bf16x8_scaled(u32x2{lo, hi}, s));
}

// ln sum_j e^(s_j) of a row from its scores' reference m (to base 2) and the
// sum of 2^(s - m); -inf of a row that sees nothing.
__device__ __forceinline__ void put_lse(const AttnLse& p, long long row, int h, float m, float sum) {
  p.lse[row * p.n_q + h] = (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// Block ids of the positions whose K, and whose V, a lane loads in a step.
struct Ids {
  int k, v;
};

// Few query rows: one row tile per workgroup (and split), whose W waves take
// the steps in turn, codes straight from the cache to registers.  The bound
// is the cache's bytes: 16 columns of the matrix instructions are there
// anyway.  A step's K codes make way for the next step's as soon as the
// scores are there, its V codes after the second product, so a wave has
// loads in flight all the time without a second set of registers.
//
// Positions are dealt so that no value ever changes lanes: a K load's lane
// (c, g) holds dimensions 16g.. of position 16(c/4) + 4t + c%4 of the step, so
// the score tile t comes out with lane (c, g) holding positions
// 16g + 4t + (0..3) of query row c -- the 16 positions whose V codes of one
// dimension are the lane's 16-byte V load, which makes the weights the B
// operand as they stand.
//
// Measured (whole calls, joins included): one sequence of 1,024 positions,
// head_dim 64, 5.7 us, of which a launch is 2.7 and the rest three loads in a
// row and one step; 16 sequences of 512 to 4,096 12.5 us (38 MB; whole
// contexts on 128 CUs, bound by what a CU takes in: codes of two steps ahead,
// and weights formed for the rows that are there alone, changed nothing); one
// of 32,768, head_dim 128, 18 us (67 MB, 13.5 us and 4.6 for the join); 3 to 6
// tokens each of 16 sequences of 700 to 8,191 37 us (148 MB, 32 and 5); 64
// sequences of 4,096, head_dim 64, 52 us (268 MB, 5.1 TB/s).  Streaming as many
// bytes without any work takes 7, 12, 27 and 48 us here.
template <int D, int W, bool LSE>
struct RowsLds {
  float lo[W][ROWS][D + 4];
  float lm[W][ROWS], ls[W][ROWS];
  float le[LSE ? W : 1][ROWS];
};

template <int D, int W, class P>
__device__ __forceinline__ void rows_item(const P& p, int item, void* smem) {
  constexpr int KH = D / 64, DT = D / 16;  // 64-dimension halves of K, 16-dimension tiles of V
  constexpr bool SCORED = Has<P>::scores, LSE = Has<P>::lse;
  typedef RowsLds<D, W, LSE> Lds;
  Lds& lds = *static_cast<Lds*>(smem);
  auto &lm = lds.lm, &ls = lds.ls;
  auto& lo = lds.lo;
  const int lb = p.c.lb, G = p.group, off = (1 << lb) - 1;
  const int head = item % p.c.n_kv;
  Item it;
  if (!find_split<FEW>(p, item / p.c.n_kv, it)) return;
  const Seq& s = it.s;
  const int l = (int)(threadIdx.x & 63u), wv = wave_id();
  const int c = l & 15, g = l >> 4;  // this lane's query row; its 16 positions of a step
  RowTile rows = row_tile(s, G, it.rt, ROWS);
  const int r0 = it.rt * ROWS;
  const bool mine = c < rows.n_rows;
  const int rr = mine ? r0 + c : r0, tok = rr / G, hd = head * G + rr % G;
  int shut = 0, see = mine ? min(max(s.pos0 + tok + 1, 0), s.len) : 0;  // this row sees [shut, see)
  float slope = 0.f;
  if constexpr (SCORED) {
    const Sight v = sight(p.b, p.x, s, tok);
    Bounds b;
    if (mine) b.add(v);
    b.join();
    rows = RowTile{rows.n_rows, b.from, b.shut, b.any, b.all};
    shut = v.lo, see = mine ? v.hi : 0;
    if (p.x.slopes) slope = slope_of(p.x.slopes[hd]);
  }
  const int t00 = rows.from / TILE, tiles = (rows.any + TILE - 1) / TILE - t00;
  const int t0 = t00 + it.step(it.split, tiles), t1 = t00 + it.step(it.split + 1, tiles);

  // Table entries of a step, loaded a step before the codes they lead to and
  // checked only there: the loads are waited for in the order of their issue,
  // so an entry asked for behind codes would arrive behind them.
  const int* row = p.b.table + (long long)s.i * p.b.width;
  const auto ids = [&](int t) {
    const int top = min((t1 * TILE - 1) >> lb, p.b.width - 1);  // the last entry that this item may need
    return Ids{row[min((t * TILE + 16 * (c >> 2)) >> lb, top)], row[min((t * TILE + 16 * g) >> lb, top)]};
  };
  // (a run of 16 that no row sees is as good as missing: its block may never have been written)
  const auto there = [&](int id, int pos) { return pos < s.len && id >= 0 && id < p.c.n_blocks && (!SCORED || pos + 16 > rows.from); };
  const unsigned bytes = (unsigned)(p.c.n_kv * D) << lb;  // of K or V of one block, all heads
  const uint8_t *kb = p.c.k + ((long long)head * D << lb), *vb = p.c.v + ((long long)head * D << lb);
  const float *ksb = p.c.ks + head, *vsb = p.c.vs + head;
  u32x4 kw[4][KH], vw[DT];
  float ks = 1.f, vs = 1.f;
  bool gone = true;  // the lane's 16 positions of V and the scores are missing
  const auto load_k = [&](int t, int id) {
    const int pk = t * TILE + 16 * (c >> 2);
    // block 0 in a missing block's place, masked later
    const unsigned ik = there(id, pk) ? (unsigned)id : 0u;
    const uint8_t* kp = kb + ((unsigned long long)ik * bytes + (unsigned)(((pk & off) + (c & 3)) * D + 16 * g));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) kw[i][h] = *reinterpret_cast<const u32x4*>(kp + 4 * i * D + 64 * h);
    ks = ksb[(unsigned long long)ik * (unsigned)p.c.n_kv];
  };
  const auto load_v = [&](int t, int id) {
    const int pv = t * TILE + 16 * g;
    gone = !there(id, pv);
    const unsigned iv = gone ? 0u : (unsigned)id;
    const uint8_t* vp = vb + ((unsigned long long)iv * bytes + (unsigned)((c << lb) + (pv & off)));
    // block 0 may never have been written: its scale must not turn 0 into NaN
    vs = vsb[(unsigned long long)iv * (unsigned)p.c.n_kv];
    vs = gone ? 1.f : vs;
#pragma unroll
    for (int d = 0; d < DT; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + ((16 * d) << lb));
  };

  const int begin = t0 + wv;
  Ids next{-1, -1}, after{-1, -1};
  if (begin < t1) {
    next = ids(begin);
    after = ids(begin + W);
  }
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
  // the weights' reference of row c (or -inf), it negated (or 0), and what the
  // lane's scores may reach before it is raised
  float m = -INFINITY, below = 0.f, up = -INFINITY, sum = 0.f, ex = 0.f;  // ex: of the weights as they are, for the log-sum-exp

  // Both are waited for here: left to itself, the second would be asked for
  // behind the first codes, and the loop's waits be for everything.
  asm volatile("" : "+v"(next.k), "+v"(next.v), "+v"(after.k), "+v"(after.v));
  if (begin < t1) {
    load_k(begin, next.k);
    load_v(begin, next.v);
    next = after;
  }
  // The last step is code of its own: behind loads that may not have been
  // issued, every wait would have to be for all of them.
  const auto step = [&](int t, auto more) {
    const int pv = t * TILE + 16 * g;
    f32x4 sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[i] = mfma16(codes_bf16(kw[i][h][2 * e], kw[i][h][2 * e + 1], ks), qv[2 * h + e], sc[i]);
    }
    if constexpr (more.value) {
      after = ids(t + 2 * W);
      load_k(t + W, next.k);
    }
    // scores of positions pv + 4i + j of row c
    // less the row's reference from the start (SCORED), but for biased ones: of far
    // positions the reference is their bias, and beside it near ones would be rounded
    float base = below;
    if constexpr (SCORED) base = p.x.slopes ? 0.f : below;
    if constexpr (SCORED) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = sc[i / 4][i % 4];
      const int rel = pv - (s.pos0 + tok);
      score<16>(p.x, p.scale, slope, base, x, [&](int i) { return rel + i; });
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i / 4][i % 4] = x[i];
    }
    if ((t + 1) * TILE > rows.all || (SCORED && t * TILE < rows.shut) || __any(gone)) {
      // opaque: a branch for the few steps that need it, not its selects in every step
      const int lim = opaque_v(gone ? 0 : see - pv), lol = SCORED ? opaque_v(shut - pv) : 0;
      const auto in = [&](int i) { return i < lim && (!SCORED || i >= lol); };
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][j] = in(4 * i + j) ? sc[i][j] : -INFINITY;
      // A NaN in V must not reach the rows that do not see it (0 * NaN): it
      // is taken out here, and put into the rows that do see it.
      uint32_t bad = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= nan_bytes(vw[d][i]);
      if (__builtin_expect(__any(bad), 0)) {
        bf16x8 seen[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i) seen[e][i] = (__bf16)(in(8 * e + i) ? 1.f : 0.f);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4 hit = f32x4{0.f, 0.f, 0.f, 0.f};
          u32x4 is;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t n = nan_bytes(vw[d][i]) >> 7;  // 1 in each NaN byte
            is[i] = n * 0x38u;                             // e4m3 of 1
            vw[d][i] &= ~(n * 0xffu);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) hit = mfma16(codes_bf16(is[2 * e], is[2 * e + 1], 1.f), seen[e], hit);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = hit[i] > 0.f ? NAN : o[d][i];
        }
      }
    }
    float mt = sc[0][0];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mt = fmaxf(mt, sc[i][j]);
    mt = SCORED ? mt - base : mt * p.scale;
    const bool rise = __any(mt > up);
    if (rise) {  // joined over the row's four lanes only here
      const float mn = fmaxf(m, max_xor32(max_xor16(mt))), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      below = mn == -INFINITY ? 0.f : -mn;
      up = mn + RISE;
      sum *= al;
      if constexpr (LSE) ex *= al;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= al;
    }
    if constexpr (SCORED) {
      if (rise || p.x.slopes) {
        const float d = below - base;
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[i] += d;
      }
    }
    float pr[16];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pr[4 * i + j] = __builtin_amdgcn_exp2f(SCORED ? sc[i][j] : fmaf(sc[i][j], p.scale, below));
      }
    if constexpr (LSE) {
#pragma unroll
      for (int i = 0; i < 16; ++i) ex += pr[i];
    }
    const bf16x2 one = bf16x2{(__bf16)1.f, (__bf16)1.f};
    bf16x8 pb[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const bf16x2 w = __builtin_convertvector(f32x2{pr[8 * e + i], pr[8 * e + i + 1]}, bf16x2);
        sum = __builtin_amdgcn_fdot2_f32_bf16(w, one, sum, false);  // of the rounded weights
        pb[e][i] = w[0];
        pb[e][i + 1] = w[1];
      }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) o[d] = mfma16(codes_bf16(vw[d][2 * e], vw[d][2 * e + 1], vs), pb[e], o[d]);
    if constexpr (more.value) {
      load_v(t + W, next.v);
      next = after;
    }
  };
  if (begin < t1) {
    int t = begin;
    for (; t + W < t1; t += W) step(t, Bool<true>{});
    step(t, Bool<false>{});
  }

  sum = sum_xor32(sum_xor16(sum));
  if constexpr (LSE) ex = sum_xor32(sum_xor16(ex));

  // join the waves: o[d][i] is dimension 16d + 4g + i of row c
  if (mine) {
    if (g == 0) lm[wv][c] = m, ls[wv][c] = sum;
    if constexpr (LSE) {
      if (g == 0) lds.le[wv][c] = ex;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&lo[wv][c][16 * d + 4 * g]) = o[d];
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < rows.n_rows * (D / 4); i += W * kWave) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float mm = lm[0][row];
#pragma unroll
    for (int w = 1; w < W; ++w) mm = fmaxf(mm, lm[w][row]);
    const float mref = mm == -INFINITY ? 0.f : mm;
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
    float tot = 0.f, te = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(lm[w][row] - mref);
      tot += f * ls[w][row];
      if constexpr (LSE) te += f * lds.le[w][row];
      v += f * *reinterpret_cast<const f32x4*>(&lo[w][row][d]);
    }
    const int tk = (r0 + row) / G, oh = head * G + (r0 + row) % G;
    if constexpr (LSE) {
      if (d == 0) {
        if (it.ns == 1) put_lse(p, s.row0 + tk, oh, mm, te);
        else p.ex[FEW][((long long)(it.slot + it.split) * p.c.n_kv + head) * ROWS + row] = te;
      }
    }
    if (it.ns == 1) {
      v *= tot > 0.f || tot != tot ? 1.f / tot : 0.f;
      uint16_t* op = static_cast<uint16_t*>(p.out.p) + (s.row0 + tk) * p.out.ts + oh * p.out.hs + d;
      u32x2 w;
      w.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, bf16x2));
      w.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, bf16x2));
      *reinterpret_cast<u32x2*>(op) = w;
    } else {
      const long long at = ((long long)(it.slot + it.split) * p.c.n_kv + head) * ROWS + row;
      *reinterpret_cast<f32x4*>(p.d[FEW].part + at * D + d) = v;
      if (d == 0) p.d[FEW].ml[at] = make_float2(mm, tot);
    }
  }
}

// Many query rows.  128 rows per workgroup, 32 to each of its four waves, on
// v_mfma_f32_32x32x16_bf16; a step's 64 positions are turned from codes to
// bf16 once and staged in LDS for all four (two buffers, one barrier a step;
// the next step's codes are in flight meanwhile).  1,024 tokens of 16 / 8 heads
// of 128 at the end of 32,768 positions: 289 us with the join's 13, 935
// TFLOP/s, where a large bf16 product reaches 1,370.  The matrix units are busy
// 40 % of the time and the vector units, mostly with the weights, as much; two
// workgroups per CU overlap them in part.  64 rows per wave (half the LDS
// reads) took 350 us: one wave per SIMD does not hide its own staging.  Without
// a past the longest tile decides, a step a microsecond: ragged prompts of 33
// to 2,048 tokens, head_dim 64, 49 us, one of 4,096 83.  Rows of LDS are padded by
// 16 bytes, which spreads the eight lanes that a 16-byte read serves at once
// over all banks.  K rows lie in LDS in the order that makes a lane's 16
// scores of 32 positions two runs of eight positions, 8h + 16m of half-wave h,
// the B operand of the second product as they stand.
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int D>
struct TileLds {
  static constexpr int KS = D + 8, VS = TILE + 8;  // row strides
  uint16_t k[2][TILE * KS];
  uint16_t v[2][D * VS];
  unsigned long long nans[2][D];  // positions of a step whose V is NaN, by dimension
  int bad[2];                     // 1 + the step in the buffer, if nans has any
};

template <int D, class P>
__device__ __forceinline__ void tile_item(const P& p, int item, void* smem) {
  constexpr bool SCORED = Has<P>::scores, LSE = Has<P>::lse;
  constexpr int KC = D / 16, DB = D / 32;    // 16-dimension pieces of a K row, 32-dimension blocks of V
  constexpr int NL = D * TILE / (256 * 16);  // 16-byte loads per thread of K, and of V
  typedef TileLds<D> Lds;
  constexpr int KS = Lds::KS, VS = Lds::VS;
  Lds& lds = *static_cast<Lds*>(smem);
  const int lb = p.c.lb, G = p.group, off = (1 << lb) - 1;
  const int head = item % p.c.n_kv;
  Item it;
  // The last items first: a prompt's last row tiles have the most positions.
  // Of several prompts the last sequence's tiles start first, whatever its
  // length (prompts of 33 to 2,048 tokens ascending / shuffled / descending:
  // head_dim 64 54 / 56 / 57 us, 128 84 / 86 / 96).
  if (!find_split<MANY>(p, p.d[MANY].items - 1 - item / p.c.n_kv, it)) return;
  const Seq& s = it.s;
  const int l = (int)(threadIdx.x & 63u), wv = wave_id(), tid = (int)threadIdx.x;
  const int c = l & 31, h = l >> 5;
  RowTile rows = row_tile(s, G, it.rt, TILE_ROWS);
  const int r0 = it.rt * TILE_ROWS;
  const bool mine = 32 * wv + c < rows.n_rows;
  const int rr = mine ? r0 + 32 * wv + c : r0, tok = rr / G, hd = head * G + rr % G;
  int shut = 0, see = mine ? min(max(s.pos0 + tok + 1, 0), s.len) : 0;  // this row sees [shut, see)
  // every row of the wave sees [none, all)
  int none = 0, all = min(max(s.pos0 + (r0 + min(32 * wv, rows.n_rows - 1)) / G + 1, 0), s.len);
  float slope = 0.f;
  if constexpr (SCORED) {
    const Sight v = sight(p.b, p.x, s, tok);
    Bounds mb, b;  // of the wave's rows, of the tile's
    if (mine) mb.add(v);
    mb.join();
    none = mb.shut, all = mb.all;
    for (int i = l; i < rows.n_rows; i += kWave) b.add(sight(p.b, p.x, s, (r0 + i) / G));
    b.join();
    rows = RowTile{rows.n_rows, b.from, b.shut, b.any, b.all};
    shut = v.lo, see = mine ? v.hi : 0;
    if (p.x.slopes) slope = slope_of(p.x.slopes[hd]);
  }
  const int t00 = rows.from / TILE, tiles = (rows.any + TILE - 1) / TILE - t00;
  const int t0 = t00 + it.step(it.split, tiles), t1 = t00 + it.step(it.split + 1, tiles);
  const int n = t1 - t0, end = min(s.len, t1 * TILE);

  bf16x8 qv[KC];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(p.q.p) + (s.row0 + tok) * p.q.ts + hd * p.q.hs + 8 * h;
#pragma unroll
    for (int k = 0; k < KC; ++k) qv[k] = *reinterpret_cast<const bf16x8*>(qp + 16 * k);
  }
  // The staging is dealt so that what a wave loads at once lies in one run of
  // 16 positions: one block, one scale, an address that is the wave's but for
  // an offset that never changes.  K: positions kt + 256 / KC * i of a step,
  // 16 dimensions; V: run wv, dimensions l and l + 64.
  const int kt = tid / KC;
  const unsigned ko = (unsigned)((kt & 15) * D + tid % KC * 16), vo = (unsigned)(l << lb);
  const unsigned bytes = (unsigned)(p.c.n_kv * D) << lb;  // of K or V of one block, all heads
  const uint8_t *kb = p.c.k + ((long long)head * D << lb), *vb = p.c.v + ((long long)head * D << lb);
  const float *ksb = p.c.ks + head, *vsb = p.c.vs + head;
  // Block ids of 16 steps, a run of 16 positions to each lane, and of the next
  // 16 in the other of two; a bit for each run that is there.
  const int* row = p.b.table + (long long)s.i * p.b.width;
  const int top = min(max(end - 1, 0) >> lb, p.b.width - 1);
  int tab0 = 0, tab1 = 0;
  unsigned long long ok0 = 0, ok1 = 0;
  const auto first_of = [&](int k) { return (t0 + k) * TILE; };
  const auto window = [&](int w) {  // looks up the runs of steps 16w .. 16w + 15
    const int pos = first_of(16 * w) + 16 * l;
    return row[min(pos >> lb, top)];
  };
  const auto confirm = [&](int w, int& tab) {  // which of them are there; the others' place is taken by block 0
    const bool ok = first_of(16 * w) + 16 * l < end && tab >= 0 && tab < p.c.n_blocks;
    tab = ok ? tab : 0;
    return __ballot(ok);
  };
  const auto id_of = [&](int k, int run) {
    const int at = (k & 15) * 4 + run;
    return (unsigned)__builtin_amdgcn_readlane(k & 16 ? tab1 : tab0, at);
  };
  const auto gone_of = [&](int k) { return ~(unsigned)((k & 16 ? ok1 : ok0) >> ((k & 15) * 4)) & 15u; };
  u32x4 kw[NL], vw[NL];
  float ks[NL], vs;
  const auto load_k = [&](int k) {
    const int first = first_of(k);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int run = (wv * (256 / KC / 4) + i * (256 / KC)) >> 4;
      const unsigned id = id_of(k, run);
      const uint8_t* base = kb + ((unsigned long long)id * bytes + (unsigned)(((first + 16 * run) & off & ~15) * D));
      kw[i] = *reinterpret_cast<const u32x4*>(base + ko);
      ks[i] = ksb[(unsigned long long)id * (unsigned)p.c.n_kv];
    }
  };
  const auto load_v = [&](int k) {
    const unsigned id = id_of(k, wv);
    const uint8_t* base = vb + ((unsigned long long)id * bytes + (unsigned)((first_of(k) + 16 * wv) & off));
#pragma unroll
    for (int i = 0; i < NL; ++i) vw[i] = *reinterpret_cast<const u32x4*>(base + (64u << lb) * i + vo);
    vs = vsb[(unsigned long long)id * (unsigned)p.c.n_kv];
  };
  const auto stage_k = [&](int k) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int j = kt + i * (256 / KC);
      // position 32a + 16m + 8h + 4b + e goes to row 32a + 16m + 8b + 4h + e
      const int r = (j & ~12) | (j & 8) >> 1 | (j & 4) << 1;
      u32x4* w = reinterpret_cast<u32x4*>(&lds.k[k & 1][r * KS + tid % KC * 16]);
      w[0] = fp8x8_to_bf16x8_scaled(u32x2{kw[i][0], kw[i][1]}, ks[i]);
      w[1] = fp8x8_to_bf16x8_scaled(u32x2{kw[i][2], kw[i][3]}, ks[i]);
    }
  };
  const auto stage_v = [&](int k) {
    const int first = first_of(k);
    if (first + TILE > rows.all || (SCORED && first < rows.shut) || gone_of(k)) {
      const int left = gone_of(k) >> wv & 1 ? 0 : opaque_v(end - first - 16 * wv);  // of the run's 16 positions
      // What no row may see is zero.  Where rows differ in what they see, a
      // NaN must not reach those that do not see it (0 * NaN): it is taken
      // out and its place noted.
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        uint32_t at = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int y = left - 4 * j;
          vw[i][j] &= y >= 4 ? 0xffffffffu : y <= 0 ? 0u : (1u << (8 * y)) - 1u;
          const uint32_t nn = nan_bytes(vw[i][j]) >> 7;  // 1 in each NaN byte
          at |= nn * 0x10204080u >> 28 << (4 * j);
          vw[i][j] &= ~(nn * 0xffu);
        }
        reinterpret_cast<uint16_t*>(&lds.nans[k & 1][l + i * 64])[wv] = (uint16_t)at;
        any |= at;
      }
      if (any) lds.bad[k & 1] = k + 1;
      vs = left <= 0 ? 1.f : vs;  // block 0's scale may be anything
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      u32x4* x = reinterpret_cast<u32x4*>(&lds.v[k & 1][(l + i * 64) * VS + 16 * wv]);
      x[0] = fp8x8_to_bf16x8_scaled(u32x2{vw[i][0], vw[i][1]}, vs);
      x[1] = fp8x8_to_bf16x8_scaled(u32x2{vw[i][2], vw[i][3]}, vs);
    }
  };

  f32x16 o[DB], sc[2];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -INFINITY, below = 0.f, up = -INFINITY, sum = 0.f, ex = 0.f;  // as in rows_item()
  // Both halves in turn: a product that adds to the one before it waits twice
  // as long as the unit takes.
  const auto scores = [&](int k) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[a][i] = 0.f;
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int a = 0; a < 2; ++a)
        sc[a] = mfma32(*reinterpret_cast<const bf16x8*>(&lds.k[k & 1][(32 * a + c) * KS + 16 * j + 8 * h]), qv[j], sc[a]);
  };

  const auto half_scores = [&](int k, int a) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[a][i] = 0.f;
#pragma unroll
    for (int j = 0; j < KC; ++j)
      sc[a] = mfma32(*reinterpret_cast<const bf16x8*>(&lds.k[k & 1][(32 * a + c) * KS + 16 * j + 8 * h]), qv[j], sc[a]);
  };

  // Step k's scores are there when its turn comes; its turn is: V of step
  // k + 1 to bf16, the weights, step k + 1's scores, the product with V, K of
  // step k + 2 to bf16.  What is staged was asked for a turn before.
  if (tid < 2) lds.bad[tid] = 0;
  if (n > 0) {
    tab0 = window(0);
    // of the first step's runs those that no row sees are as good as missing: their blocks may never have been written
    if constexpr (SCORED) tab0 = first_of(0) + 16 * l + 16 > rows.from ? tab0 : -1;
    tab1 = window(1);
    ok0 = confirm(0, tab0);
    ok1 = confirm(1, tab1);
    load_k(0);
    load_v(0);
  }
  // q is waited for here: inside the loop the wait would stand in every step,
  // behind the next step's codes
#pragma unroll
  for (int k = 0; k < KC; ++k) asm volatile("" : "+v"(qv[k]));
  __syncthreads();
  if (n > 0) {
    stage_k(0);
    load_k(1);
    stage_v(0);
  }
  __syncthreads();
  if (n > 0) {
    scores(0);
    stage_k(1);
    load_k(2);
    load_v(1);
  }
  __syncthreads();

  for (int k = 0; k < n; ++k) {
    const int first = first_of(k), buf = k & 1;
    const unsigned gone = gone_of(k);
    // window w + 1, looked up and confirmed during window w, in the place of w - 1
    if ((k & 15) == 12 && k > 16) {
      if (k & 16) ok0 = confirm((k >> 4) + 1, tab0);
      else ok1 = confirm((k >> 4) + 1, tab1);
    }
    stage_v(k + 1);
    load_v(k + 2);
    if ((k & 15) == 1 && k > 16) {
      const int x = window((k >> 4) + 1);
      if (k & 16) tab0 = x;
      else tab1 = x;
    }
    float base = below;  // as in rows_item()
    if constexpr (SCORED) base = p.x.slopes ? 0.f : below;
    // score i of half a: position 32a + 16(i/8) + 8h + i%8 of the step
    const auto place = [](int a, int i) { return 32 * a + 16 * (i / 8) + i % 8; };
    if constexpr (SCORED) {
      const int rel = first + 8 * h - (s.pos0 + tok);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = sc[a][i];
        score<16>(p.x, p.scale, slope, base, x, [&](int i) { return rel + place(a, i); });
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[a][i] = x[i];
      }
    }
    if (first + TILE > all || (SCORED && first < none) || gone) {
      // opaque: a branch for the few steps that need it, not its 64 selects in every step
      const int lim = opaque_v(see - first - 8 * h), lol = SCORED ? opaque_v(shut - first - 8 * h) : 0;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sc[a][i] = place(a, i) < lim && (!SCORED || place(a, i) >= lol) && !(gone >> (2 * a + i / 8) & 1) ? sc[a][i] : -INFINITY;
    }
    float mt = sc[0][0];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, sc[a][i]);
    mt = SCORED ? mt - base : mt * p.scale;
    const bool rise = __any(mt > up);
    if (rise) {
      const float mn = fmaxf(m, max_xor32(mt)), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      below = mn == -INFINITY ? 0.f : -mn;
      up = mn + RISE;
      sum *= al;
      if constexpr (LSE) ex *= al;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= al;
    }
    if constexpr (SCORED) {
      if (rise || p.x.slopes) {
        const float d = below - base;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[a][i] += d;
      }
    }
    if (__builtin_expect((first + TILE > rows.all || (SCORED && first < rows.shut) || gone) && lds.bad[buf] == k + 1, 0)) {
      // the NaN that stage_v() took out, put into the rows that see them
      const int x = min(max(see - first, 0), TILE);
      unsigned long long seen = x < 64 ? (1ull << x) - 1ull : ~0ull;
      if constexpr (SCORED) {
        const int y = min(max(shut - first, 0), TILE);
        seen &= y < 64 ? ~0ull << y : 0ull;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) seen &= gone >> i & 1 ? ~(0xffffull << (16 * i)) : ~0ull;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (lds.nans[buf][32 * d + 8 * (i / 4) + 4 * h + i % 4] & seen) o[d][i] = NAN;
    }
    const bf16x2 one = bf16x2{(__bf16)1.f, (__bf16)1.f};
    bf16x8 pb[2][2];
    const auto weights = [&](int a) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float x = __builtin_amdgcn_exp2f(SCORED ? sc[a][i] : fmaf(sc[a][i], p.scale, below));
        const float y = __builtin_amdgcn_exp2f(SCORED ? sc[a][i + 1] : fmaf(sc[a][i + 1], p.scale, below));
        if constexpr (LSE) ex += x + y;
        const bf16x2 w = __builtin_convertvector(f32x2{x, y}, bf16x2);
        sum = __builtin_amdgcn_fdot2_f32_bf16(w, one, sum, false);  // of the rounded weights
        pb[a][i / 8][i % 8] = w[0];
        pb[a][i / 8][i % 8 + 1] = w[1];
      }
    };
    const auto add_v = [&](int a) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < DB; ++d)
          o[d] = mfma32(*reinterpret_cast<const bf16x8*>(&lds.v[buf][(32 * d + c) * VS + 32 * a + 16 * i + 8 * h]), pb[a][i], o[d]);
    };
    weights(0);
    if constexpr (SCORED) {
      // a half's weights beside the other's products (16 / 8 heads of 64, four
      // prompts of 2,048 72 us; in the order below 76)
      half_scores(k + 1, 0);
      add_v(0);
      weights(1);
      half_scores(k + 1, 1);
      add_v(1);
    } else {
      weights(1);
      scores(k + 1);  // of the last step, of nothing: not used
      add_v(0);
      add_v(1);
    }
    stage_k(k + 2);
    load_k(k + 3);
    __syncthreads();
  }
  sum = sum_xor32(sum);
  if constexpr (LSE) {
    ex = sum_xor32(ex);
    if (mine && h == 0) {
      if (it.ns == 1) put_lse(p, s.row0 + tok, hd, m, ex);
      else p.ex[MANY][((long long)(it.slot + it.split) * p.c.n_kv + head) * TILE_ROWS + 32 * wv + c] = ex;
    }
  }
  if (!mine) return;
  // o[d][4b + j] is dimension 32d + 8b + 4h + j of row c
  if (it.ns == 1) {
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    uint16_t* op = static_cast<uint16_t*>(p.out.p) + (s.row0 + tok) * p.out.ts + hd * p.out.hs + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x2 w;
        w.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[d][4 * b] * inv, o[d][4 * b + 1] * inv}, bf16x2));
        w.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{o[d][4 * b + 2] * inv, o[d][4 * b + 3] * inv}, bf16x2));
        *reinterpret_cast<u32x2*>(op + 32 * d + 8 * b) = w;
      }
  } else {
    const long long at = ((long long)(it.slot + it.split) * p.c.n_kv + head) * TILE_ROWS + 32 * wv + c;
    float* pp = p.d[MANY].part + at * D + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<f32x4*>(pp + 32 * d + 8 * b) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    if (h == 0) p.d[MANY].ml[at] = make_float2(m, sum);
  }
}

template <int D, int W, class P>
__global__ __launch_bounds__(W* kWave, D == 64 ? 3 : 2) void attn_rows(P p) {
  __shared__ __align__(16) RowsLds<D, W, Has<P>::lse> lds;
  rows_item<D, W>(p, (int)blockIdx.x, &lds);
}
template <int D, class P>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_tile(P p) {
  __shared__ __align__(16) TileLds<D> lds;
  tile_item<D>(p, (int)blockIdx.x, &lds);
}
// Batches with sequences of both kinds: one launch, so that neither waits for
// the other's last workgroup; the tiles first, they take longest.
template <int D, class P>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_both(P p) {
  __shared__ __align__(16) union {
    TileLds<D> t;
    RowsLds<D, 4, Has<P>::lse> r;
  } lds;
  const int many = p.d[MANY].items * p.c.n_kv;
  if ((int)blockIdx.x < many) tile_item<D>(p, (int)blockIdx.x, &lds);
  else rows_item<D, 4>(p, (int)blockIdx.x - many, &lds);
}

// Where a row's partials are.
struct Parts {
  const float* part;  // the first split's outputs
  const float2* ml;
  long long stride;   // rows from one split to the next
};
template <int D>
__device__ __forceinline__ Parts parts_of(const Attn& p, const Item& it, int oh) {
  const Deal& d = p.d[it.kind];
  const long long r = (long long)it.rt * p.group + oh % p.group, rt = r >> d.lr;
  Parts x;
  x.stride = (long long)p.c.n_kv << d.lr;
  const long long at = (((it.slot + rt * it.ns) * p.c.n_kv + oh / p.group) << d.lr) + r - (rt << d.lr);
  x.part = d.part + at * D;
  x.ml = d.ml + at;
  return x;
}
__device__ __forceinline__ const float* ex_of(const AttnLse& p, const Item& it, const Parts& x) {
  return p.ex[it.kind] + (x.ml - p.d[it.kind].ml);
}
__device__ __forceinline__ void put_row4(const Rows& out, long long e, f32x4 a, float tot) {
  a *= tot > 0.f || tot != tot ? 1.f / tot : 0.f;
  u32x2 w;
  w.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a[0], a[1]}, bf16x2));
  w.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a[2], a[3]}, bf16x2));
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out.p) + e) = w;
}

// Joins the splits of the rows that have more than one; D/4 lanes read a
// partial, the order of the sums is fixed.  Many rows: a wave takes HEADS
// rows of one token after the other.
template <int D, int HEADS, class P>
__global__ __launch_bounds__(256) void attn_join_waves(P p) {
  constexpr int LPP = D / 4, NG = kWave / LPP, PER = 8;  // lanes per partial, partials at once, loads in flight
  const int l = (int)(threadIdx.x & 63u), per_token = (p.n_q + HEADS - 1) / HEADS;
  const int w = (int)blockIdx.x * 4 + wave_id();
  Item it;
  if (!find_split<-1>(p, w / per_token, it) || it.ns == 1) return;
  const int ns = it.ns, ln = l % LPP, grp = l / LPP, h0 = w % per_token * HEADS;
  for (int oh = h0; oh < min(h0 + HEADS, p.n_q); ++oh) {
    const Parts x = parts_of<D>(p, it, oh);
    float mm = -INFINITY;
    for (int z = l; z < ns; z += kWave) mm = fmaxf(mm, x.ml[z * x.stride].x);
    mm = wave_max(mm);
    const float mref = mm == -INFINITY ? 0.f : mm;
    float tot = 0.f;
    f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int z0 = grp; z0 < ns; z0 += PER * NG) {
      f32x4 v[PER];
      float2 q[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int z = z0 + i * NG;
        q[i] = z < ns ? x.ml[z * x.stride] : make_float2(-INFINITY, 0.f);
        v[i] = z < ns ? *reinterpret_cast<const f32x4*>(x.part + z * x.stride * D + 4 * ln) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float f = __builtin_amdgcn_exp2f(q[i].x - mref);
        tot += f * q[i].y;
        a += f * v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (NG == 4) a[i] = sum_xor16(a[i]);
      a[i] = sum_xor32(a[i]);
    }
    if (NG == 4) tot = sum_xor16(tot);
    tot = sum_xor32(tot);
    if (grp == 0) put_row4(p.out, (it.s.row0 + it.rt) * p.out.ts + oh * p.out.hs + 4 * ln, a, tot);
    if constexpr (Has<P>::lse) {
      float te = 0.f;
      for (int z = l; z < ns; z += kWave) te += __builtin_amdgcn_exp2f(x.ml[z * x.stride].x - mref) * ex_of(p, it, x)[z * x.stride];
      te = wave_sum(te);
      if (l == 0) put_lse(p, it.s.row0 + it.rt, oh, mm, te);
    }
  }
}

// Few rows: a workgroup for each, 64 partials in flight together (one sequence
// of 32,768, head_dim 128, in a graph 18.9 us; with 32 19.8).  5 us, of which a launch
// is 2.7 and the rest the lengths, the partials and the sums in turn.
template <int D, class P>
__global__ __launch_bounds__(256) void attn_join(P p) {
  constexpr int LPP = D / 4, NG = 256 / LPP, PER = 64 / NG;  // lanes per partial, groups, partials in flight per group
  __shared__ float lw[kMaxSplits], red1[4];
  __shared__ f32x4 red[NG][LPP];
  const int oh = (int)(blockIdx.x % (unsigned)p.n_q);
  Item it;
  if (!find_split<-1>(p, (int)(blockIdx.x / (unsigned)p.n_q), it)) return;
  const int ns = it.ns;
  if (ns == 1) return;
  const Parts x = parts_of<D>(p, it, oh);
  const int ln = (int)threadIdx.x % LPP, grp = (int)threadIdx.x / LPP, tz = (int)threadIdx.x;
  f32x4 v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int z = grp + i * NG;
    v[i] = z < ns ? *reinterpret_cast<const f32x4*>(x.part + z * x.stride * D + 4 * ln) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float2 q = tz < ns ? x.ml[tz * x.stride] : make_float2(-INFINITY, 0.f);
  const float mm = block_max<4>(q.x, red1);
  const float w = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(q.x - mm);
  lw[tz] = w;
  const float tot = block_sum<4>(w * q.y, red1);
  if constexpr (Has<P>::lse) {
    const float te = block_sum<4>(tz < ns ? w * ex_of(p, it, x)[tz * x.stride] : 0.f, red1);
    if (tz == 0) put_lse(p, it.s.row0 + it.rt, oh, mm, te);
  }
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PER; ++i) a += lw[grp + i * NG] * v[i];
  for (int z = grp + PER * NG; z < ns; z += NG) a += lw[z] * *reinterpret_cast<const f32x4*>(x.part + z * x.stride * D + 4 * ln);
  red[grp][ln] = a;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < NG; ++i) a += red[i][ln];
    put_row4(p.out, (it.s.row0 + it.rt) * p.out.ts + oh * p.out.hs + 4 * ln, a, tot);
  }
}

}  // namespace kv8
}  // namespace mk
