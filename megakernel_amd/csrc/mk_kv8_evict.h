// Eviction from the paged 8-bit KV cache by accumulated attention weight
// (kv8.hip has the host side): weigh() adds up what each cached position got,
// choose() finds the heaviest positions of a sequence and KV head, move() takes
// them to blocks of their own.  No atomics on memory: every sum has one owner
// and a fixed order.
#pragma once
#include "mk_kv8.h"

namespace mk {
namespace kv8 {

struct Mass {
  float* p;
  long long ss, hs;  // elements from one sequence / KV head to the next
};

// ------------------------------------------------------------------- weigh
// mass[j] = (j before the batch's rows ? mass[j] : 0) + sum over rows r and the
// heads that share the KV head of e^(s_rj - lse_r).
struct Weigh {
  Cache c;
  Batch b;
  Rows q;
  const float* lse;
  Mass mass;
  int n_q, group;
  float scale;  // softmax scale * log2(e)
  Scores x;
};

// Sum over the 16 lanes of a row of each of 16 values; lane c gets value c's.
// Partners of every step hold the same values: mirrored lanes first.
__device__ __forceinline__ float scatter_sum(float (&v)[16], int c) {
  const auto half = [&](auto ctrl, auto n, int bit) {
    constexpr int N = decltype(n)::value;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float keep = bit ? v[i + N] : v[i], give = bit ? v[i] : v[i + N];
      v[i] = keep + dpp_sel<decltype(ctrl)::value>(give);
    }
  };
  half(Int<DPP_MIRROR>{}, Int<8>{}, c & 8);
  half(Int<DPP_HALF_MIRROR>{}, Int<4>{}, c & 4);
  half(Int<DPP_XOR2>{}, Int<2>{}, c & 2);
  half(Int<DPP_XOR1>{}, Int<1>{}, c & 1);
  return v[0];
}

// A wave holds the K of 64 positions of one KV head and goes through the query
// rows, 16 at a time, on v_mfma_f32_16x16x32_bf16 (the positions' layout is
// that of rows_item()); its weights stay in 16 sums a lane until the end.
// Few rows: every wave has positions of its own.  Many (SPLIT): the W waves of
// a workgroup share the positions and deal the row tiles.
template <int D, int W, bool SPLIT>
__global__ __launch_bounds__(W* kWave) void weigh(Weigh p) {
  constexpr int KH = D / 64;
  __shared__ float red[SPLIT ? W : 1][TILE];
  const int lb = p.c.lb, G = p.group, off = (1 << lb) - 1;
  const int l = (int)(threadIdx.x & 63u), wv = wave_id(), c = l & 15, g = l >> 4;
  const unsigned n_kv = (unsigned)p.c.n_kv;
  const int head = (int)(blockIdx.x % n_kv), stride = (int)(gridDim.x / n_kv) * (SPLIT ? 1 : W);
  const unsigned bytes = (unsigned)(p.c.n_kv * D) << lb;
  for (int it = (int)(blockIdx.x / n_kv) * (SPLIT ? 1 : W) + (SPLIT ? 0 : wv);; it += stride) {
    Seq s;
    int t;
    if (!find_item(p.b, lb, it, [&](const Seq& q) { return q.rows > 0 ? (q.len + TILE - 1) / TILE : 0; }, s, t)) return;
    const int first = t * TILE, n_rows = s.rows * G;
    const int* row = p.b.table + (long long)s.i * p.b.width;
    const auto there = [&](int pos) {
      if (pos >= s.len) return -1;
      const int id = row[pos >> lb];
      return id >= 0 && id < p.c.n_blocks ? id : -1;
    };
    const int pk = first + 16 * (c >> 2);
    const int idk = there(pk), idv = there(first + 16 * g);
    u32x4 kw[4][KH];
    const unsigned ik = idk < 0 ? 0u : (unsigned)idk;
    const uint8_t* kp = p.c.k + ((long long)head * D << lb) + ((unsigned long long)ik * bytes + (unsigned)(((pk & off) + (c & 3)) * D + 16 * g));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) kw[i][h] = *reinterpret_cast<const u32x4*>(kp + 4 * i * D + 64 * h);
    const float ks = p.c.ks[(unsigned long long)ik * n_kv + head];
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    // without a prefix the rows before these positions do not see them
    int r0 = 0;
    if (!(p.x.prefix && p.x.prefix[s.i] > first)) r0 = (int)min(max(((long long)first - s.pos0) * G, 0ll), (long long)n_rows) & ~15;
    for (r0 += SPLIT ? 16 * wv : 0; r0 < n_rows; r0 += SPLIT ? 16 * W : 16) {
      const bool mine = r0 + c < n_rows;
      const int rr = mine ? r0 + c : r0, tok = rr / G, hd = head * G + rr % G;
      Sight v = sight(p.b, p.x, s, tok);
      if (!mine) v = Sight{0, 0};
      if (!__any(v.lo < first + TILE && v.hi > first)) continue;
      const uint16_t* qp = static_cast<const uint16_t*>(p.q.p) + (s.row0 + tok) * p.q.ts + hd * p.q.hs;
      bf16x8 qv[2 * KH];
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) qv[2 * h + e] = *reinterpret_cast<const bf16x8*>(qp + 64 * h + 16 * g + 8 * e);
      const float ref = p.lse[(long long)(s.row0 + tok) * p.n_q + hd] * 1.4426950408889634f;
      const float slope = p.x.slopes ? p.x.slopes[hd] * 1.4426950408889634f : 0.f;
      float sc[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < KH; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) a = mfma16(codes_bf16(kw[i][h][2 * e], kw[i][h][2 * e + 1], ks), qv[2 * h + e], a);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[4 * i + j] = a[j];
      }
      const int pv = first + 16 * g, rel = pv - (s.pos0 + tok);
      score<16>(p.x, p.scale, slope, sc, [&](int i) { return rel + i; });
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(sc[i] - ref);
      if (__any(v.lo > first || v.hi < first + TILE || idv < 0)) {
        const int lim = opaque_v(idv < 0 ? 0 : v.hi - pv), lol = opaque_v(v.lo - pv);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = i < lim && i >= lol ? sc[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += sc[i];
    }
    float sum = scatter_sum(acc, c);
    if constexpr (SPLIT) {
      __syncthreads();  // the sums of the positions before are read
      red[wv][l] = sum;
      __syncthreads();
      if (wv) continue;
      sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += red[w][l];
    }
    const int pos = first + l;
    if (pos < s.len) {
      float* m = p.mass.p + s.i * p.mass.ss + head * p.mass.hs + pos;
      *m = pos < s.pos0 ? *m + sum : sum;
    }
  }
}

// ------------------------------------------------------------------ choose
struct Choose {
  Mass mass;
  const int* len;
  int* kept;
  int* kept_len;
  int n_kv, keep, recent, sinks, positions;
};

// Weights as integers of the same order: NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);
  return w != w ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}

// Bits of m below this lane's.
__device__ __forceinline__ unsigned lanes_below(unsigned long long m) {
  return (unsigned)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
}

// One workgroup per sequence and KV head.  The smallest key that stays is
// found digit by digit (11, 11 and 10 bits) from counts in LDS; each wave then
// writes the positions of its own stretch in order.
__global__ __launch_bounds__(1024) void choose(Choose p) {
  constexpr int NW = 16, BINS = 2048;
  __shared__ unsigned hist[BINS], part[NW], found[2];
  __shared__ unsigned above[NW], same[NW];
  const int tid = (int)threadIdx.x, l = tid & 63, wv = wave_id();
  const int i = (int)(blockIdx.x / (unsigned)p.n_kv), head = (int)(blockIdx.x % (unsigned)p.n_kv);
  const int len = min(max(p.len[i], 0), p.positions);
  int* kept = p.kept + (long long)blockIdx.x * p.keep;
  const int m = min(len, p.keep);
  if (head == 0 && tid == 0) p.kept_len[i] = m;
  if (len <= p.keep) {
    for (int j = tid; j < p.keep; j += 1024) kept[j] = j < m ? j : -1;
    return;
  }
  const float* w = p.mass.p + i * p.mass.ss + head * p.mass.hs;
  const int a = p.sinks, e = len - p.recent, want = p.keep - p.sinks - p.recent;  // `want` of [a, e)
  for (int j = tid; j < p.sinks; j += 1024) kept[j] = j;
  for (int j = tid; j < p.recent; j += 1024) kept[p.keep - p.recent + j] = e + j;
  if (want == 0) return;
  const int n = e - a, seg = (n + NW * 64 - 1) / (NW * 64) * 64;  // positions of a wave
  const int j0 = a + wv * seg, j1 = min(j0 + seg, e);
  uint32_t prefix = 0, mask = 0;
  unsigned left = (unsigned)want;  // to find among the keys that match the prefix
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int b = tid; b < BINS; b += 1024) hist[b] = 0;
    __syncthreads();
    for (int j = j0 + l; j < j1; j += 64) {
      const uint32_t k = key_of(w[j]);
      if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // from the highest digit down: thread t has digits 2047 - 2t and the one below
    const unsigned h0 = hist[BINS - 1 - 2 * tid], h1 = hist[BINS - 2 - 2 * tid];
    const unsigned up = (unsigned)wave_prefix((int)(h0 + h1));
    if (l == 63) part[wv] = up;
    __syncthreads();
    unsigned before = up - (h0 + h1);
    for (int k = 0; k < wv; ++k) before += part[k];
    if (before < left && left <= before + h0) found[0] = BINS - 1 - 2 * tid, found[1] = before;
    else if (before + h0 < left && left <= before + h0 + h1) found[0] = BINS - 2 - 2 * tid, found[1] = before + h0;
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= ((1u << bits) - 1) << shift;
    left -= found[1];
  }
  // keys above `prefix` stay, and the first `left` that equal it
  unsigned na = 0, ns = 0;
  for (int j = j0; j < j1; j += 64) {
    const uint32_t k = j + l < j1 ? key_of(w[j + l]) : 0;
    na += (unsigned)__popcll(__ballot(j + l < j1 && k > prefix));
    ns += (unsigned)__popcll(__ballot(j + l < j1 && k == prefix));
  }
  if (l == 0) above[wv] = na, same[wv] = ns;
  __syncthreads();
  unsigned ba = 0, bs = 0;
  for (int k = 0; k < wv; ++k) ba += above[k], bs += same[k];
  for (int j = j0; j < j1; j += 64) {
    const bool in = j + l < j1;
    const uint32_t k = in ? key_of(w[j + l]) : 0;
    const unsigned long long ma = __ballot(in && k > prefix), ms = __ballot(in && k == prefix);
    const unsigned ra = ba + lanes_below(ma), rs = bs + lanes_below(ms);
    if (in && (k > prefix || (k == prefix && rs < left))) kept[a + ra + min(rs, left)] = j + l;
    ba += (unsigned)__popcll(ma);
    bs += (unsigned)__popcll(ms);
  }
}

// -------------------------------------------------------------------- move
struct Move {
  Cache c;
  const int* table;      // the blocks that are read, [n_seq][width]
  const int* kept;       // [n_seq][n_kv][keep]
  const int* kept_len;
  const int* new_table;  // those that are written, [n_seq][new_width]
  int width, new_width, keep;
  Mass from, to;
};

// One team of T threads per new block and head, in append()'s pieces of 4 rows
// x 8 dimensions.  A new block's scale is the smallest that fits its rows;
// codes are rounded again where it is larger than the one they come from.
template <int D, int T, int PASSES>
__global__ __launch_bounds__(256) void move(Move p) {
  constexpr int HEADS = 256 / T;
  __shared__ float red[4][2];
  const unsigned sets = (unsigned)((p.c.n_kv + HEADS - 1) / HEADS), per = (unsigned)(p.keep + (1 << p.c.lb) - 1) >> p.c.lb;
  const unsigned it = blockIdx.x / sets;
  const int i = (int)(it / per), j = (int)(it % per), lb = p.c.lb, B = 1 << lb;
  const int tid = (int)threadIdx.x, head = (int)(blockIdx.x % sets) * HEADS + tid / T;
  const int m = min(min(max(p.kept_len[i], 0), p.keep), (int)min((long long)p.new_width << lb, 0x7fffffffll));
  const int p0 = j << lb, rows = min(m - p0, B);
  if (rows <= 0) return;
  const int to = p.new_table[(long long)i * p.new_width + j];
  const bool on = head < p.c.n_kv && to >= 0 && to < p.c.n_blocks;
  const int* kept = p.kept + ((long long)i * p.c.n_kv + min(head, p.c.n_kv - 1)) * p.keep + p0;
  const int* table = p.table + (long long)i * p.width;
  u32x2 kw[PASSES][4];
  uint32_t vw[PASSES][8];  // V's dwords of the new block: byte r is row r of the piece
  int ek[PASSES][4], ev[PASSES][4];
  float kmax = 0.f, vmax = 0.f;
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    const Piece pc = piece_at<D, 8>(tid % T + q * T, lb);
#pragma unroll
    for (int d = 0; d < 8; ++d) vw[q][d] = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      kw[q][r] = u32x2{0, 0};
      ek[q][r] = ev[q][r] = -126;
      const int at = on && pc.row + r < rows ? kept[pc.row + r] : -1;
      if (at < 0 || at >> lb >= p.width) continue;
      const int id = table[at >> lb];
      if (id < 0 || id >= p.c.n_blocks) continue;
      const long long src = (long long)id * p.c.n_kv + head;
      kw[q][r] = *reinterpret_cast<const u32x2*>(p.c.k + (src * D << lb) + (at & (B - 1)) * D + pc.dim);
      const uint8_t* vp = p.c.v + ((src * D + pc.dim) << lb) + (at & (B - 1));
#pragma unroll
      for (int d = 0; d < 8; ++d) vw[q][d] |= (uint32_t)vp[d << lb] << (8 * r);
      const float ks = p.c.ks[src], vs = p.c.vs[src];
      ek[q][r] = ks > 0.f ? max(min(ilogbf(ks), 127), -126) : -126;
      ev[q][r] = vs > 0.f ? max(min(ilogbf(vs), 127), -126) : -126;
    }
  }
  // the largest value: of a row the largest magnitude among its codes, NaN left out
#pragma unroll
  for (int q = 0; q < PASSES; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float f[4], a = 0.f, b = 0.f;
      const float ks = ldexpf(1.f, ek[q][r]), vs = ldexpf(1.f, ev[q][r]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        decode4(kw[q][r][h], 1.f, f);
#pragma unroll
        for (int x = 0; x < 4; ++x) a = fmaxf(a, fabsf(f[x]));
        decode4(gather4(vw[q][4 * h], vw[q][4 * h + 1], vw[q][4 * h + 2], vw[q][4 * h + 3], r), 1.f, f);
#pragma unroll
        for (int x = 0; x < 4; ++x) b = fmaxf(b, fabsf(f[x]));
      }
      kmax = fmaxf(kmax, a * ks);
      vmax = fmaxf(vmax, b * vs);
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
    for (int x = 0; x < T / 64; ++x) kmax = fmaxf(kmax, red[w + x][0]), vmax = fmaxf(vmax, red[w + x][1]);
  }
  if (head < p.c.n_kv && p.to.p) {
    for (int r = tid % T; r < rows; r += T) {
      const int at = kept[r];
      const bool is = at >= 0 && at >> lb < p.width;
      p.to.p[i * p.to.ss + head * p.to.hs + p0 + r] = is ? p.from.p[i * p.from.ss + head * p.from.hs + at] : 0.f;
    }
  }
  if (!on) return;
  const int ke = scale_exp(kmax), ve = scale_exp(vmax);
  const long long dst = (long long)to * p.c.n_kv + head;
  if (tid % T == 0) {
    p.c.ks[dst] = ldexpf(1.f, ke);
    p.c.vs[dst] = ldexpf(1.f, ve);
  }
  uint8_t *kd = p.c.k + (dst * D << lb), *vd = p.c.v + (dst * D << lb);
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    const Piece pc = piece_at<D, 8>(tid % T + q * T, lb);
    const int n = min(rows - pc.row, 4);  // rows of the piece
    if (n <= 0) continue;
    float vr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // a code that is not zero is at most 448 of the new scale, so its scale is at most 2^18 of it
      const float kr = ldexpf(1.f, min(ek[q][r] - ke, 30));
      vr[r] = ldexpf(1.f, min(ev[q][r] - ve, 30));
      if (r < n) *reinterpret_cast<u32x2*>(kd + (pc.row + r) * D + pc.dim) = u32x2{rescale4(kw[q][r].x, kr), rescale4(kw[q][r].y, kr)};
    }
    const uint32_t keep = n < 4 ? 0xffffffffu << (8 * n) : 0u;  // bytes of rows behind the last
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      float f[4];
      decode4(vw[q][d], 1.f, f);
      uint32_t x = encode4(f[0] * vr[0], f[1] * vr[1], f[2] * vr[2], f[3] * vr[3]);
      uint32_t* w = reinterpret_cast<uint32_t*>(vd + ((pc.dim + d) << lb) + pc.row);
      if (keep) x = (x & ~keep) | (*w & keep);
      *w = x;
    }
  }
}

}  // namespace kv8
}  // namespace mk
