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

// A step of N positions of a sequence.
struct Step {
  Seq s;
  int first;
};
template <int N>
__device__ __forceinline__ bool find_step(const Weigh& p, int it, Step& r) {
  int t;
  if (!find_item(p.b, p.c.lb, it, [](const Seq& q) { return q.rows > 0 ? (q.len + N - 1) / N : 0; }, r.s, t)) return false;
  r.first = t * N;
  return true;
}
// Block of a position that is there, or -1.
__device__ __forceinline__ int block_at(const Weigh& p, const Seq& s, int pos) {
  return pos < s.len ? block_id(p.b, s.i, pos >> p.c.lb, p.c.n_blocks) : -1;
}
// Tokens from here on see position `first` (without a prefix, which earlier ones see too).
__device__ __forceinline__ int first_token(const Weigh& p, const Step& x) {
  if (p.x.prefix && p.x.prefix[x.s.i] > x.first) return 0;
  return (int)min(max((long long)x.first - x.s.pos0, 0ll), (long long)x.s.rows);
}

// Few rows: a wave holds the K of 64 positions and goes through the query rows,
// 16 at a time, on v_mfma_f32_16x16x32_bf16 (the positions' layout is that of
// rows_item()); its weights stay in 16 sums a lane until the end.  Bound by K's way
// here: one token to each of 16 sequences of 512 to 4,096, head_dim 64 (19 MB of K),
// takes 9.0 us, of which 2.7 are the launch and the rest three loads in a row;
// 16 of 4,096, 4 tokens each, 12.4, head_dim 128 22 (67 MB, 3.1 TB/s).
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 3) void weigh_few(Weigh p) {
  constexpr int KH = D / 64;
  const int lb = p.c.lb, G = p.group, off = (1 << lb) - 1;
  const int l = (int)(threadIdx.x & 63u), c = l & 15, g = l >> 4;
  const unsigned n_kv = (unsigned)p.c.n_kv;
  const int head = (int)(blockIdx.x % n_kv), stride = (int)(gridDim.x / n_kv) * 4;
  const unsigned bytes = (unsigned)(p.c.n_kv * D) << lb;
  for (int it = (int)(blockIdx.x / n_kv) * 4 + wave_id();; it += stride) {
    Step x;
    if (!find_step<TILE>(p, it, x)) return;
    const Seq& s = x.s;
    const int first = x.first, n_rows = s.rows * G, pos = first + l;
    float* mass = p.mass.p + s.i * p.mass.ss + head * p.mass.hs + pos;
    const float was = pos < min(s.len, s.pos0) ? *mass : 0.f;
    const int pk = first + 16 * (c >> 2), pv = first + 16 * g;
    const int idk = block_at(p, s, pk), idv = block_at(p, s, pv);
    const unsigned ik = idk < 0 ? 0u : (unsigned)idk;
    const uint8_t* kp = p.c.k + ((long long)head * D << lb) + ((unsigned long long)ik * bytes + (unsigned)(((pk & off) + (c & 3)) * D + 16 * g));
    u32x4 kw[4][KH];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) kw[i][h] = *reinterpret_cast<const u32x4*>(kp + 4 * i * D + 64 * h);
    const float ks = p.c.ks[(unsigned long long)ik * n_kv + head];
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int r0 = (int)min((long long)first_token(p, x) * G, (long long)n_rows) & ~15; r0 < n_rows; r0 += 16) {
      const bool mine = r0 + c < n_rows;
      const int rr = mine ? r0 + c : r0, tok = rr / G, hd = head * G + rr - tok * G;
      Sight v = sight(p.b, p.x, s, tok);
      if (!mine) v = Sight{0, 0};
      if (!__any(v.lo < first + TILE && v.hi > first)) continue;
      const uint16_t* qp = static_cast<const uint16_t*>(p.q.p) + (s.row0 + tok) * p.q.ts + hd * p.q.hs + 16 * g;
      bf16x8 qv[2 * KH];
#pragma unroll
      for (int h = 0; h < 2 * KH; ++h) qv[h] = *reinterpret_cast<const bf16x8*>(qp + 64 * (h / 2) + 8 * (h % 2));
      const float ref = p.lse[(long long)(s.row0 + tok) * p.n_q + hd] * 1.4426950408889634f;
      const float slope = p.x.slopes ? slope_of(p.x.slopes[hd]) : 0.f;
      float sc[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2 * KH; ++h) a = mfma16(codes_bf16(kw[i][h / 2][2 * (h % 2)], kw[i][h / 2][2 * (h % 2) + 1], ks), qv[h], a);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[4 * i + j] = a[j];
      }
      const int rel = pv - (s.pos0 + tok);
      score<16>(p.x, p.scale, slope, -ref, sc, [&](int i) { return rel + i; });
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(sc[i]);
      if (__any(v.lo > first || v.hi < first + TILE || idv < 0)) {
        const int lim = opaque_v(idv < 0 ? 0 : v.hi - pv), lol = opaque_v(v.lo - pv);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = i < lim && i >= lol ? sc[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += sc[i];
    }
    const float sum = scatter_sum(acc, c);
    if (pos < s.len) *mass = was + sum;
  }
}

// Many rows: a wave holds the K of 32 positions as bf16 and goes through the rows,
// up to 32 at a time, on v_mfma_f32_32x32x16_bf16.  A tile is whole tokens (of more
// than 32 heads, 32 heads of one).  Its q comes row by row straight into LDS that is
// the wave's own (no barriers), the next tile's while this one's weights are formed.
// (Into registers each of a row's 16-byte pieces is asked for by itself, the waves'
// tiles do not fit the L1, and q comes several times.)  The eight waves of a
// workgroup are PS side by side, which ask for the same tiles at about the same
// time, and 8 / PS groups that deal the rows.  Sums stay in 16 registers a lane, and
// meet over lanes and groups, in a fixed order, at the end.
// 1,024 tokens of 16 / 8 heads of 128 at the end of 16,384 positions take 121 us (one
// side by side 130), capped 151; 1,024 tokens without a past 20 (14, capped 17).
// What bounds it is q's way from the L2 (a tile for every 1,024 scores) beside the
// vector unit, which one wave alone can give an operation only every eight cycles:
// positions are so few that four waves fit a SIMD.
template <int D, int PS>
__global__ __launch_bounds__(512, 4) void weigh_many(Weigh p) {
  constexpr int W = 8, N = 32, RS = W / PS;           // waves, positions of each, groups of rows
  constexpr int KC = D / 16, CH = D / 8, NL = CH / 2;  // products' depth, 16-byte pieces of a row, loads of a lane
  __shared__ __align__(512) u32x4 tile[W][32 * CH];
  __shared__ long long off[32 * CH];  // of each 16 bytes of a tile, from its first row: bytes
  __shared__ float red[RS][PS * N];
  const int lb = p.c.lb, G = p.group;
  const int l = (int)(threadIdx.x & 63u), wv = wave_id(), ps = wv % PS, rg = wv / PS, c = l & 31, h = l >> 5;
  const unsigned n_kv = (unsigned)p.c.n_kv;
  const int head = (int)(blockIdx.x % n_kv), stride = (int)(gridDim.x / n_kv);
  const unsigned bytes = (unsigned)(p.c.n_kv * D) << lb;
  const int per = G <= 32 ? 32 / G : 1, sets = (G + 31) / 32;  // tokens of a tile, tiles of a token
  const int dt = G <= 32 ? c / G : 0, dh = c - dt * G;         // the lane's token and head in it
  // Piece k of row r lies at k ^ (r % CH): a column's reads are spread over all
  // banks.  Rows past a tile's tokens are the first row again.
  for (int i = (int)threadIdx.x; i < 32 * CH; i += W * kWave) {
    const int r = i / CH, t = G <= 32 ? r / G : 0;
    off[i] = (t < per && t < p.b.n_tokens ? 2 * (t * p.q.ts + (r - t * G) * p.q.hs) : 0) + 16 * ((i ^ r) & (CH - 1));
  }
  __syncthreads();
  const char* q0 = static_cast<const char*>(p.q.p) + 2ll * head * G * p.q.hs;
  typedef const __attribute__((address_space(3))) bf16x8* LdsRow;
  const unsigned mine0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) u32x4*)&tile[wv][c * CH] + 16u * ((2 * h) ^ (c & (CH - 1)));
  for (int it = (int)(blockIdx.x / n_kv);; it += stride) {
    Step x;
    if (!find_step<PS * N>(p, it, x)) return;
    const Seq& s = x.s;
    const int begin = x.first;
    const int first = x.first += ps * N;
    // position first + c; its dimensions 32j + 16h .. of K row and q row alike
    const int at = first + c, id = block_at(p, s, first + (c & 16));
    const unsigned ik = id < 0 ? 0u : (unsigned)id;
    const uint8_t* kp = p.c.k + ((long long)head * D << lb) + ((unsigned long long)ik * bytes + (unsigned)((at & ((1 << lb) - 1)) * D + 16 * h));
    const float ks = p.c.ks[(unsigned long long)ik * n_kv + head];
    const unsigned long long no = __ballot(id < 0);
    const unsigned gone = ((unsigned)no & 1u) | ((unsigned)(no >> 15) & 2u);  // runs of 16 positions that are not there
    bf16x8 ka[KC];
#pragma unroll
    for (int j = 0; j < KC / 2; ++j) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(kp + 32 * j);
      ka[2 * j] = codes_bf16(w[0], w[1], ks);
      ka[2 * j + 1] = codes_bf16(w[2], w[3], ks);
    }
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    struct Rows32 {
      int u, first, set;  // the tile's first token among all, and first head
      int tok;
      float lse, slope;
      Sight v;
    };
    int t1 = (s.rows + per - 1) / per;
    if (p.x.window) {  // tokens further on see none of these
      const long long last = (long long)first + N + p.x.window - 1 - s.pos0;
      t1 = (int)min((long long)t1, (max(last, 0ll) + per - 1) / per);
    }
    const int units = t1 * sets;
    // The first tile from y.u on of which some row sees some of the positions,
    // and its q on the way.
    const auto fetch = [&](Rows32& y) {
      for (; y.u < units; y.u += RS) {
        const int t = sets == 1 ? y.u : y.u / sets, set = 32 * (y.u - t * sets);
        // so that all 32 rows are there; rows of the tile before do not count again
        y.first = max(min(s.row0 + t * per, p.b.n_tokens - per), 0);
        y.set = max(min(set, G - 32), 0);
        y.tok = y.first + dt - s.row0;
        const bool mine = dt < per && y.tok >= t * per && y.tok < s.rows && y.set + dh >= set;
        y.tok = mine ? y.tok : t * per;
        y.v = mine ? sight(p.b, p.x, s, y.tok) : Sight{0, 0};
        if (!__any(y.v.lo < first + N && y.v.hi > first)) continue;
        const char* qp = q0 + 2 * ((long long)y.first * p.q.ts + (long long)y.set * p.q.hs);
        // all of them before the first load: a read of LDS waits for loads into it
        long long at[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) at[i] = off[64 * i + l];
#pragma unroll
        for (int i = 0; i < NL; ++i)
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(qp + at[i]),
                                           (__attribute__((address_space(3))) void*)&tile[wv][64 * i], 16, 0, 0);
        const int hd = head * G + (mine ? y.set + dh : 0);
        y.lse = p.lse[(long long)(s.row0 + y.tok) * p.n_q + hd];
        y.slope = p.x.slopes ? p.x.slopes[hd] : 0.f;  // (nothing here waits for it)
        return true;
      }
      return false;
    };
    Rows32 y;
    y.u = first_token(p, x) / per * sets + rg;
    bool more = first < s.len && fetch(y);
    while (more) {
      const float ref = y.lse * 1.4426950408889634f, slope = slope_of(y.slope);
      const Sight v = y.v;
      const int rel = first + 4 * h - (s.pos0 + y.tok);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // q is in LDS
      const unsigned row = (unsigned)opaque_v((int)mine0);  // piece 2h of row c; k pieces on is 16k ^ that
      f32x16 sc;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j)
        sc = mfma32(ka[j], *(LdsRow)(uintptr_t)(row ^ (16u * (4 * (j / 2) + j % 2))), sc);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and has been read: the next may come
      y.u += RS;
      more = fetch(y);
      // score i: position 8(i/4) + 4h + i%4
      float e[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = sc[i];
      score<16>(p.x, p.scale, slope, -ref, e, [&](int i) { return rel + 8 * (i / 4) + i % 4; });
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(e[i]);
      if (__any(v.lo > first || v.hi < first + N) || gone) {
        const int lim = opaque_v(v.hi - first - 4 * h), lol = opaque_v(v.lo - first - 4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 8 * (i / 4) + i % 4;
          e[i] = j < lim && j >= lol && !(gone >> (i / 8) & 1) ? e[i] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += e[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = sum_xor16(acc[i]);
    const float sum = scatter_sum(acc, c & 15);  // of position 8(i/4) + 4h + i%4, i = c % 16
    __syncthreads();                             // the sums of the positions before are read
    red[rg][ps * N + 8 * (c % 16 / 4) + 4 * h + c % 4] = sum;
    __syncthreads();
    if (wv == 0 && l < PS * N && begin + l < s.len) {
      float* mass = p.mass.p + s.i * p.mass.ss + head * p.mass.hs + begin + l;
      float all = red[0][l];
#pragma unroll
      for (int r = 1; r < RS; ++r) all += red[r][l];
      *mass = begin + l < s.pos0 ? *mass + all : all;
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
  const int b = __float_as_int(w + 0.f);
  return w != w ? 0u : (uint32_t)(b ^ (b >> 31 | (int)0x80000000));
}

// Bits of m below this lane's.
__device__ __forceinline__ unsigned lanes_below(unsigned long long m) {
  return (unsigned)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
}

// One workgroup per sequence and KV head.  The smallest key that stays is
// found digit by digit, eight bits each, from counts in LDS; each wave then
// writes the positions of its own stretch in order.  Weights share few
// exponents, and lanes that count the same wait for each other, so the counts of
// a digit are in COPIES by lane.  Up to PER * 1,024 candidates stay in LDS, each wave's own; of
// more every look reads them again.  (In registers every loop over them is
// straight code of 32 turns, and fetching that took longer than running it:
// 8,192 candidates 15.7 us, here 10.)  32,768 candidates take 19 us, 4,096 7.5: a CU's
// vector units are at them all the time, some 60 operations for every 64.
template <int PER>
__global__ __launch_bounds__(1024) void choose(Choose p) {
  constexpr int NW = 16, COPIES = 16, U = 4;
  __shared__ u32x4 hist[256 * COPIES / 4];
  __shared__ uint32_t keys[PER * 1024];
  __shared__ unsigned part[NW], found[2], above[NW], same[NW];
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
  // looks of a wave, 64 positions each; U at a time, so that their waits are one
  const int n = e - a, seg = (n + NW * 64 * U - 1) / (NW * 64 * U) * U;
  const int j0 = a + wv * seg * 64 + l, looks = want ? min(seg, (max(n - wv * seg * 64, 0) + 64 * U - 1) / (64 * U) * U) : 0;
  // Past the last candidate a key is 0, the lowest: its positions come last, so
  // it is found only where more are wanted than there are.
  // (Loads are never skipped, or each would be waited for by itself.)
  const auto load = [&](int y) { return w[min(j0 + 64 * y, e - 1)]; };
  const auto key = [&](int y, float x) { return j0 + 64 * y < e ? key_of(x) : 0u; };
  uint32_t* mine = keys + wv * PER * 64 + l;
  const bool kept_keys = seg <= PER;
  // every look of the wave at its 64 positions: f(position, key)
  const auto each = [&](auto f) {
    if (kept_keys) {
      for (int y = 0; y < looks; y += U) {
        uint32_t k[U];
#pragma unroll
        for (int x = 0; x < U; ++x) k[x] = mine[64 * (y + x)];
#pragma unroll
        for (int x = 0; x < U; ++x) f(j0 + 64 * (y + x), k[x]);
      }
    } else {
      for (int y = 0; y < looks; y += U) {
        float v[U];
#pragma unroll
        for (int x = 0; x < U; ++x) v[x] = load(y + x);
#pragma unroll
        for (int x = 0; x < U; ++x) f(j0 + 64 * (y + x), key(y + x, v[x]));
      }
    }
  };
  for (int j = tid; j < p.sinks; j += 1024) kept[j] = j;
  for (int j = tid; j < p.recent; j += 1024) kept[p.keep - p.recent + j] = e + j;
  if (want == 0) return;
  unsigned* count = reinterpret_cast<unsigned*>(hist) + (unsigned)l % COPIES;
  hist[tid] = u32x4{0, 0, 0, 0};
  __syncthreads();
  // the first digit's counts as the keys arrive
  if (kept_keys) {
    constexpr int N = PER < 16 ? PER : 16;
    for (int y = 0; y < looks; y += N) {  // past its own looks a wave writes what nothing reads
      float v[N];
#pragma unroll
      for (int x = 0; x < N; ++x) v[x] = load(y + x);
      uint32_t k[N];
      if (a + (wv * seg + y + N) * 64 <= e) {
#pragma unroll
        for (int x = 0; x < N; ++x) k[x] = key_of(v[x]);
      } else {
#pragma unroll
        for (int x = 0; x < N; ++x) k[x] = key(y + x, v[x]);
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        mine[64 * (y + x)] = k[x];
        if (y + x < looks) atomicAdd(count + (k[x] >> 24) * COPIES, 1u);
      }
    }
  } else {
    each([&](int, uint32_t k) { atomicAdd(count + (k >> 24) * COPIES, 1u); });
  }
  uint32_t prefix = 0;
  unsigned left = (unsigned)want;  // to find among the keys that match the prefix
#pragma unroll
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (shift < 24) {
      hist[tid] = u32x4{0, 0, 0, 0};
      __syncthreads();
      each([&](int, uint32_t k) {
        if ((k ^ prefix) < 1u << (shift + 8) % 32) atomicAdd(count + (k >> shift & 255u) * COPIES, 1u);
      });
    }
    __syncthreads();
    // from the highest digit down, four threads to a digit
    const u32x4 v = hist[1023 - tid];
    unsigned h = v[0] + v[1] + v[2] + v[3];
    h += (unsigned)__builtin_amdgcn_update_dpp(0, (int)h, DPP_XOR1, 0xf, 0xf, true);
    h += (unsigned)__builtin_amdgcn_update_dpp(0, (int)h, DPP_XOR2, 0xf, 0xf, true);
    const unsigned up = (unsigned)wave_prefix(l % 4 ? 0 : (int)h);
    if (l == 63) part[wv] = up;
    __syncthreads();
    unsigned before = up - h;
#pragma unroll
    for (int k = 0; k < NW; ++k) before += k < wv ? part[k] : 0;
    if (l % 4 == 0 && before < left && left <= before + h) found[0] = (1023 - tid) / 4, found[1] = before;
    __syncthreads();
    prefix |= found[0] << shift;
    left -= found[1];
  }
  // keys above `prefix` stay, and the first `left` that equal it
  unsigned na = 0, ns = 0;
  each([&](int, uint32_t k) {
    na += (unsigned)__popcll(__ballot(k > prefix));
    ns += (unsigned)__popcll(__ballot(k == prefix));
  });
  if (l == 0) above[wv] = na, same[wv] = ns;
  __syncthreads();
  unsigned ba = 0, bs = 0;
#pragma unroll
  for (int k = 0; k < NW; ++k) ba += k < wv ? above[k] : 0, bs += k < wv ? same[k] : 0;
  each([&](int j, uint32_t k) {
    const unsigned long long ma = __ballot(k > prefix), ms = __ballot(k == prefix);
    if (!ms) {
      if (k > prefix) kept[a + (int)(ba + min(bs, left) + lanes_below(ma))] = j;
    } else {
      const unsigned ra = ba + lanes_below(ma), rs = bs + lanes_below(ms);
      if (k > prefix || (k == prefix && rs < left)) kept[a + (int)(ra + min(rs, left))] = j;
    }
    ba += (unsigned)__popcll(ma);
    bs += (unsigned)__popcll(ms);
  });
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

// Exponent of a scale as append() takes an older one.
__device__ __forceinline__ int exponent_of(float s) { return s > 0.f ? max(min(ilogbf(s), 127), -126) : -126; }
// Largest magnitude of four codes, NaN left out.
__device__ __forceinline__ float top4(uint32_t w) {
  float f[4];
  decode4(w, 1.f, f);
  return fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3])));
}

// One team of T threads per new block and head; a new block's scale is the
// smallest that fits its rows, and codes are rounded again where it is larger
// than the one they come from.  Where each row comes from is looked up once, into
// LDS.  A thread holds 16 codes of K, a piece of a row, and 16 of V, as many
// dimensions of one row: lanes are rows there, so a load's bytes lie in as few
// lines as there are old blocks among the rows (in pieces of 4 rows x 8
// dimensions every byte was a line of its own).  Four lanes then trade dimensions
// for rows, which makes the dwords of the new block.  4,096 rows of 32,768, 8 heads of
// 128, take 11 us (18 in pieces), 1,000 of each of 16 contexts of 512 to 4,096, heads of
// 64, 14 (21): four loads in a row (lengths and kept positions, table, scales, codes),
// and V's bytes one by one.
template <int D, int T, int PASSES>
__global__ __launch_bounds__(256) void move(Move p) {
  constexpr int HEADS = 256 / T, CH = D / 16;  // pieces of a K row
  constexpr int ROWS_MAX = T * PASSES / CH;    // rows of a block
  __shared__ int src[HEADS][ROWS_MAX], old[HEADS][ROWS_MAX];  // block and row, block -1 where there is none
  __shared__ int ek[HEADS][ROWS_MAX], ev[HEADS][ROWS_MAX];
  __shared__ float red[4][2];
  const unsigned sets = (unsigned)((p.c.n_kv + HEADS - 1) / HEADS), per = (unsigned)(p.keep + (1 << p.c.lb) - 1) >> p.c.lb;
  const unsigned it = blockIdx.x / sets;
  const int i = (int)(it / per), j = (int)(it % per), lb = p.c.lb, B = 1 << lb;
  const int tid = (int)threadIdx.x, h0 = (int)(blockIdx.x % sets) * HEADS, team = tid / T, head = h0 + team;
  const int m = min(min(max(p.kept_len[i], 0), p.keep), (int)min((long long)p.new_width << lb, 0x7fffffffll));
  const int p0 = j << lb, rows = min(m - p0, B);
  // asked for before the lengths are there
  static_assert(HEADS * ROWS_MAX <= 256, "a thread for every row");
  const int h = tid >> lb, r = tid & (B - 1);
  const bool own = tid < HEADS * B && h0 + h < p.c.n_kv && p0 + r < p.keep;
  const int at = own ? p.kept[((long long)i * p.c.n_kv + h0 + h) * p.keep + p0 + r] : -1;
  const int to = j < p.new_width ? p.new_table[(long long)i * p.new_width + j] : -1;
  if (rows <= 0) return;
  const bool on = head < p.c.n_kv && to >= 0 && to < p.c.n_blocks;
  if (tid < HEADS * B) {
    int s = -1, o = 0, a = -126, b = -126;
    if (own && r < rows) {
      const bool is = at >= 0 && at >> lb < p.width;
      const int id = is ? p.table[(long long)i * p.width + (at >> lb)] : -1;
      if (p.to.p) p.to.p[i * p.to.ss + (h0 + h) * p.to.hs + p0 + r] = is ? p.from.p[i * p.from.ss + (h0 + h) * p.from.hs + at] : 0.f;
      if (id >= 0 && id < p.c.n_blocks) {
        s = id, o = at & (B - 1);
        const long long w = (long long)id * p.c.n_kv + h0 + h;
        a = exponent_of(p.c.ks[w]);
        b = exponent_of(p.c.vs[w]);
      }
    }
    src[h][r] = s, old[h][r] = o, ek[h][r] = a, ev[h][r] = b;
  }
  __syncthreads();
  u32x4 kw[PASSES], vw[PASSES];
  int ke[PASSES], ve[PASSES];
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    const int u = tid % T + q * T, kr = u / CH, vr = u & (B - 1), vd = u >> lb << 4;
    kw[q] = vw[q] = u32x4{0, 0, 0, 0};
    const int a = on ? src[team][kr] : -1, b = on ? src[team][vr] : -1;
    if (a >= 0) kw[q] = *reinterpret_cast<const u32x4*>(p.c.k + ((((long long)a * p.c.n_kv + head) << lb) + old[team][kr]) * D + u % CH * 16);
    if (b >= 0) {
      const uint8_t* v = p.c.v + ((((long long)b * p.c.n_kv + head) * D + vd) << lb) + old[team][vr];
#pragma unroll
      for (int d = 0; d < 16; ++d) vw[q][d / 4] |= (uint32_t)v[d << lb] << (8 * (d % 4));
    }
    ke[q] = ek[team][kr], ve[q] = ev[team][vr];
  }
  float kmax = 0.f, vmax = 0.f;
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) a = fmaxf(a, top4(kw[q][x])), b = fmaxf(b, top4(vw[q][x]));
    kmax = fmaxf(kmax, ldexpf(a, ke[q]));
    vmax = fmaxf(vmax, ldexpf(b, ve[q]));
  }
  kmax = wave_max(kmax);
  vmax = wave_max(vmax);
  if constexpr (T > 64) {
    if (tid % 64 == 0) red[tid / 64][0] = kmax, red[tid / 64][1] = vmax;
    __syncthreads();
    const int w = tid / T * (T / 64);
#pragma unroll
    for (int x = 0; x < T / 64; ++x) kmax = fmaxf(kmax, red[w + x][0]), vmax = fmaxf(vmax, red[w + x][1]);
  }
  if (!on) return;
  const int kn = scale_exp(kmax), vn = scale_exp(vmax);
  const long long dst = (long long)to * p.c.n_kv + head;
  if (tid % T == 0) {
    p.c.ks[dst] = ldexpf(1.f, kn);
    p.c.vs[dst] = ldexpf(1.f, vn);
  }
  uint8_t *kd = p.c.k + (dst * D << lb), *vd = p.c.v + (dst * D << lb);
  // a code that is not zero is at most 448 of the new scale, so its scale is at most 2^18 of it
  const auto ratio = [](int from, int to) { return ldexpf(1.f, min(from - to, 30)); };
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    const int u = tid % T + q * T, kr = u / CH;
    const float a = ratio(ke[q], kn), b = ratio(ve[q], vn);
    if (kr < rows) {
      u32x4 x;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = rescale4(kw[q][y], a);
      *reinterpret_cast<u32x4*>(kd + (u << 4)) = x;
    }
    // dword x of the lane: dimensions 4x.. of its row; after the trade lane y of four has dimensions 4y.. of four rows
    u32x4 x;
#pragma unroll
    for (int y = 0; y < 4; ++y) x[y] = rescale4(vw[q][y], b);
    const int y = tid & 3, row = (u & (B - 1)) & ~3, dim = (u >> lb << 4) + 4 * y;
    u32x4 z;
    const auto from = [&](auto lane) {  // dword y of that lane of the four
      constexpr int L = decltype(lane)::value, CTRL = L | L << 2 | L << 4 | L << 6;
      uint32_t r = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[k], CTRL, 0xf, 0xf, true);
        r = y == k ? t : r;
      }
      return r;
    };
    z[0] = from(Int<0>{}), z[1] = from(Int<1>{}), z[2] = from(Int<2>{}), z[3] = from(Int<3>{});
    const int n = min(rows - row, 4);
    if (n <= 0) continue;
    const uint32_t keep = n < 4 ? 0xffffffffu << (8 * n) : 0u;  // bytes of rows behind the last
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t v = gather4(z[0], z[1], z[2], z[3], d);
      uint32_t* w = reinterpret_cast<uint32_t*>(vd + ((dim + d) << lb) + row);
      if (keep) v = (v & ~keep) | (*w & keep);
      *w = v;
    }
  }
}

}  // namespace kv8
}  // namespace mk
