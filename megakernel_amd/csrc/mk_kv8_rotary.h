// Rotary positions of query and key rows without a norm, in both layouts, for
// the first `turned` dimensions of a head (kv8.hip has the host side):
//   half         pairs (i, i + turned/2)
//   interleaved  pairs (2i, 2i + 1)
// (a, b) -> A (a cos t - b sin t, b cos t + a sin t), t = pos * inv_freq[i]; the
// dimensions behind are copied.  Contexts longer than trained for are a matter
// of inv_freq and of the amplitude A.
#pragma once
#include "mk_kv8.h"

namespace mk {
namespace kv8 {

struct Turn {
  Rows q, k, qo, ko;
  const float* freq;
  const int* pos;
  int n_tokens, n_q, n_kv, dim, turned;
  float amplitude;
};

// Sine and cosine of pos * freq times the amplitude.  The angle is a product
// of a 31-bit and a 24-bit number, formed and reduced to a fraction of a turn
// in fp64 (as norm_rope() does).
__device__ __forceinline__ void turn_of(double turns_per, float freq, float amplitude, float& sn, float& cs) {
  double turns = turns_per * (double)freq;
  turns -= rint(turns);
  sincospif(2.f * (float)turns, &sn, &cs);
  sn *= amplitude;
  cs *= amplitude;
}
__device__ __forceinline__ double turns_per(int pos) { return (double)pos * 0.15915494309189535; }  // turns of one radian

// A thread holds 16 elements of a head, eight whole pairs or what is copied,
// and takes HPT heads of one token with one set of sines and cosines, whose
// arithmetic would else stand beside the loads of every head.  8,192 tokens of 24
// heads of 128, half of each turned, bf16 (101 MB) take 20.4 us, 4.9 TB/s; 4,096 tokens,
// whole, fp32 to bf16 (76 MB) 15.4, 4.9 TB/s; a copy of 2 GiB reaches 4.9.  16 tokens
// 3.3 us, where an empty launch takes 2.7.
template <bool SRC32, bool DST32, bool INTERLEAVED, int HPT>
__global__ __launch_bounds__(256) void rotate(Turn p) {
  const unsigned units = (unsigned)p.dim / 16, heads = (unsigned)(p.n_q + p.n_kv), sets = (heads + HPT - 1) / HPT;
  const unsigned id = blockIdx.x * 256 + threadIdx.x;
  const unsigned rest = id / units, u = id - rest * units, t = rest / sets, set = rest - t * sets;
  if (t >= (unsigned)p.n_tokens) return;
  const bool turned = 16 * u < (unsigned)p.turned;
  const int e0 = !INTERLEAVED && turned ? 8 * u : 16 * u, e1 = !INTERLEAVED && turned ? p.turned / 2 + 8 * u : 16 * u + 8;
  float x[HPT][2][8];
  const auto rows = [&](unsigned h, const Rows& q, const Rows& k, long long& at) -> const Rows& {
    const Rows& r = h < (unsigned)p.n_q ? q : k;
    at = t * r.ts + (h < (unsigned)p.n_q ? h : h - p.n_q) * r.hs;
    return r;
  };
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const unsigned h = set + i * sets;
    if (h >= heads) break;
    long long at;
    const Rows& r = rows(h, p.q, p.k, at);
    load8<SRC32>(r.p, at + e0, x[i][0]);
    load8<SRC32>(r.p, at + e1, x[i][1]);
  }
  if (turned) {
    const double per = turns_per(p.pos[t]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float sn, cs;
      turn_of(per, p.freq[8 * u + j], p.amplitude, sn, cs);
#pragma unroll
      for (int i = 0; i < HPT; ++i) {
        float& a = INTERLEAVED ? x[i][j / 4][2 * j % 8] : x[i][0][j];
        float& b = INTERLEAVED ? x[i][j / 4][2 * j % 8 + 1] : x[i][1][j];
        const float y = a * cs - b * sn;
        b = b * cs + a * sn;
        a = y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const unsigned h = set + i * sets;
    if (h >= heads) break;
    long long at;
    const Rows& r = rows(h, p.qo, p.ko, at);
    store8<DST32>(r.p, at + e0, x[i][0]);
    store8<DST32>(r.p, at + e1, x[i][1]);
  }
}

template <bool F32>
__device__ __forceinline__ float get1(const void* p, long long e) {
  if constexpr (F32) return static_cast<const float*>(p)[e];
  else return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[e] << 16);
}
template <bool F32>
__device__ __forceinline__ void put1(void* p, long long e, float x) {
  if constexpr (F32) static_cast<float*>(p)[e] = x;
  else static_cast<__bf16*>(p)[e] = (__bf16)x;
}

// Any even sizes and any alignment: a pair to a thread, with sines of its own and
// loads of single elements (8,192 tokens of 24 heads of 128, half of each turned, rows
// one element off: 52 us, aligned 21 in rotate()).
template <bool SRC32, bool DST32>
__global__ __launch_bounds__(256) void rotate_pairs(Turn p, int interleaved) {
  const unsigned pairs = (unsigned)p.dim / 2, heads = (unsigned)(p.n_q + p.n_kv);
  const unsigned id = blockIdx.x * 256 + threadIdx.x;
  const unsigned rest = id / pairs, i = id - rest * pairs, t = rest / heads, h = rest - t * heads;
  if (t >= (unsigned)p.n_tokens) return;
  const bool is_k = h >= (unsigned)p.n_q, turned = 2 * i < (unsigned)p.turned;
  const unsigned hh = is_k ? h - p.n_q : h;
  const Rows &src = is_k ? p.k : p.q, &dst = is_k ? p.ko : p.qo;
  const int ea = turned && !interleaved ? i : 2 * i, eb = turned && !interleaved ? i + p.turned / 2 : 2 * i + 1;
  const long long s = t * src.ts + hh * src.hs, d = t * dst.ts + hh * dst.hs;
  float a = get1<SRC32>(src.p, s + ea), b = get1<SRC32>(src.p, s + eb);
  if (turned) {
    float sn, cs;
    turn_of(turns_per(p.pos[t]), p.freq[i], p.amplitude, sn, cs);
    const float y = a * cs - b * sn;
    b = b * cs + a * sn;
    a = y;
  }
  put1<DST32>(dst.p, d + ea, a);
  put1<DST32>(dst.p, d + eb, b);
}

}  // namespace kv8
}  // namespace mk
