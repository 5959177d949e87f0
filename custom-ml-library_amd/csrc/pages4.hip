// The 4-bit paged cache (pages4.h): quantising append, values read back, page
// copies and table entries.
#include "pages4.h"
#include "rope_math.h"

namespace tsattn {
namespace {

constexpr int NT = 256, NW = NT / 64;

struct RowArgs {
  Pages4 p;
  Seqs s;
  View k, v;
  const void *cos, *sin;
  int len, tiles;  // positions a sequence, tiles that they can touch at most
};

// The largest scale of a cache of T: 6 s is finite in it.
template <typename T>
constexpr float most_scale() {
  return std::is_same_v<T, f16> ? 10752.f : 1.3125f * 0x1p125f;
}

// A group's scale from the largest magnitude's bits (compared as integers, in
// which a NaN is the largest of all).  The fp32 quotient m / 6 by the reciprocal, its
// exact remainder and one correction (Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990: correctly rounded); where that
// remainder would underflow, the scale is its least value either way.
template <typename T>
__device__ __forceinline__ float scale_of(uint32_t m) {
#pragma clang fp contract(off)
  constexpr float r = 1.f / 6.f;
  const float x = __builtin_bit_cast(float, m), q0 = x * r;
  uint32_t u = __builtin_bit_cast(uint32_t, __builtin_fmaf(__builtin_fmaf(-q0, 6.f, x), r, q0));
  u = (u + 0x1FFFFu + ((u >> 18) & 1u)) & ~0x3FFFFu;  // 5 mantissa bits
  const float s = fminf(fmaxf(__builtin_bit_cast(float, u), 0x1p-27f), most_scale<T>());
  return m >= 0x7F800000u ? __builtin_nanf("") : s;
}

// The largest magnitude's bits of eight values.
template <typename T>
__device__ __forceinline__ uint32_t most_of(const u32x4 (&raw)[sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, raw[i >> 2][i & 3] & 0x7FFFFFFFu);
    return m;
  } else {  // (16-bit integers order as the values do: pairs at a time)
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    auto two = [&](int i) { return __builtin_bit_cast(u16x2, raw[0][i] & 0x7FFF7FFFu); };
    const u16x2 x = __builtin_elementwise_max(__builtin_elementwise_max(two(0), two(1)),
                                              __builtin_elementwise_max(two(2), two(3)));
    const uint16_t most = x[0] > x[1] ? x[0] : x[1];
    return __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(T, most)));
  }
}

// Eight codes.  The quotient is x / s to within an ulp's rounding: x times the
// reciprocal in two parts (45 bits), rounded once, so it is exact where x / s is half way
// between two levels.  For 16-bit x no other quotient comes that near to such a point
// (x has at most 11 significant bits, the point times s 9), so the conversion's
// rounding (to nearest, ties to even, saturating) decides as the real quotient does.
// fp32 quotients are truncated with a sticky last bit instead, so that none rounds
// onto one.  The reciprocal's low part has its bits while it is a normal number, for
// scales under 2^100: larger ones and their values come down by 2^64 first, exactly (what
// falls out of fp32 there has code 0 either way).
template <typename T>
__device__ __forceinline__ uint32_t codes_of(float (&x)[8], float s) {
#pragma clang fp contract(off)
  if constexpr (most_scale<T>() > 0x1p64f) {
    if (s > 0x1p64f) {
      s *= 0x1p-64f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= 0x1p-64f;
    }
  }
  const float rc = __builtin_amdgcn_rcpf(s), rl = __builtin_fmaf(-rc, s, 1.f) * rc;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = __builtin_fmaf(x[i], rc, x[i] * rl);
    if constexpr (std::is_same_v<T, float>) {
      const float m = fabsf(q[i]), r = __builtin_fmaf(-m, s, fabsf(x[i]));
      uint32_t u = __builtin_bit_cast(uint32_t, m);
      if (r < 0.f && u != 0u) --u;
      if (r != 0.f) u |= 1u;
      q[i] = copysignf(__builtin_bit_cast(float, u), x[i]);
    }
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.f, 3);
  return w;
}

// Largest of four neighbouring lanes.
__device__ __forceinline__ uint32_t quad_umax(uint32_t x) {
  x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0xB1, 0xF, 0xF, true)));
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x4E, 0xF, 0xF, true)));
}

// Keys' words <-> values' words.  Lane 4 g' + q (of any g) has, of channels 8 o .. + 7,
// the codes of key 4 g' + q in word a and of key 16 + 4 g' + q in word b; the quad's
// transpose gives it channels 8 o + q (in a) and 8 o + 4 + q (in b) of the quad's eight
// keys: a value word each.  Two butterflies inside the quad (codes between lanes q
// and q ^ 1, bytes between q and q ^ 2), each its own inverse, then halves.
struct Transpose {
  uint32_t m1, m2, r1, r2;
  __device__ __forceinline__ explicit Transpose(int lane)
      : m1(lane & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu), m2(lane & 2 ? 0xFF00FF00u : 0x00FF00FFu),
        r1(lane & 1 ? 4u : 28u), r2(lane & 2 ? 8u : 24u) {}
  template <int CTRL>
  __device__ __forceinline__ static uint32_t exchange(uint32_t x, uint32_t mask, uint32_t turn) {
    const uint32_t y = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, true));
    return (x & mask) | (__builtin_amdgcn_alignbit(y, y, turn) & ~mask);
  }
  __device__ __forceinline__ uint32_t codes(uint32_t x) const { return exchange<0xB1>(x, m1, r1); }  // lanes q, q ^ 1
  __device__ __forceinline__ uint32_t bytes(uint32_t x) const { return exchange<0x4E>(x, m2, r2); }  // lanes q, q ^ 2
  __device__ __forceinline__ void to_values(uint32_t &a, uint32_t &b) const {
    const uint32_t x = bytes(codes(a)), y = bytes(codes(b));
    a = __builtin_amdgcn_perm(y, x, 0x05040100u);  // low halves: the first channel, keys of x then of y
    b = __builtin_amdgcn_perm(y, x, 0x07060302u);
  }
  __device__ __forceinline__ void to_keys(uint32_t &a, uint32_t &b) const {
    const uint32_t x = __builtin_amdgcn_perm(b, a, 0x05040100u), y = __builtin_amdgcn_perm(b, a, 0x07060302u);
    a = codes(bytes(x));
    b = codes(bytes(y));
  }
};

// Where a lane's word of channel 32 ks + 8 g + 4 e + q (c = 4 g' + q) lies among the
// values' words: lane 16 g' + 8 (g & 1) + 4 e + q, word 2 ks + g / 2.
template <int G>
__device__ __forceinline__ int value_at(int c, int g, int ks, int e) {
  return word4<G>(2 * ks + (g >> 1), 16 * (c >> 2) + 8 * (g & 1) + 4 * e + (c & 3));
}

template <int G>
__device__ __forceinline__ void store_words(char *to, int lane, const uint32_t (&word)[2 * G]) {
  if constexpr (G == 1) {
    *reinterpret_cast<u32x2 *>(to + 8 * lane) = u32x2{word[0], word[1]};
  } else {
#pragma unroll
    for (int q = 0; q < G / 2; ++q)
      *reinterpret_cast<u32x4 *>(to + (64 * q + lane) * 16) =
          u32x4{word[4 * q], word[4 * q + 1], word[4 * q + 2], word[4 * q + 3]};
  }
}
template <int G>
__device__ __forceinline__ void load_words(const char *from, int lane, uint32_t (&word)[2 * G]) {
  if constexpr (G == 1) {
    const u32x2 r = *reinterpret_cast<const u32x2 *>(from + 8 * lane);
    word[0] = r[0], word[1] = r[1];
  } else {
#pragma unroll
    for (int q = 0; q < G / 2; ++q) {
      const u32x4 r = *reinterpret_cast<const u32x4 *>(from + (64 * q + lane) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) word[4 * q + i] = r[i];
    }
  }
}

// One wave quantises the new positions of one tile, head and side (keys or values).
// A load takes whole rows, PPR lanes of 8 channels a row, so that four neighbouring
// lanes make a group and the angles' loads take whole lines of their tables too (four
// 64-byte pieces a row from the operand order's lanes: 44 us where this took 38, now
// 35, 4 x 8 heads x 8192 positions of D128 in bf16, rotated: 172 MB at 4.9 TB/s, a
// large copy's rate).  Codes and scales then cross
// the wave through LDS into operand order; values' words, one channel of eight keys
// each, take a transpose in each quad of lanes and a second trip.  A tile that is
// only partly new keeps its other positions: keys' words belong to one position each,
// values' are read, merged and written.
template <typename T, int G>
__global__ __launch_bounds__(NT) void append_kernel(RowArgs a) {
  constexpr int D = 32 * G, W = 2 * G;
  constexpr int PPR = D / 8, KPI = 64 / PPR;  // pieces a row, rows a load
  constexpr int QW = sizeof(T) / 2;           // 16-byte loads a piece
  __shared__ __attribute__((aligned(16))) char lds[NW][18 * D];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x * NW + wv;  // (tile, side, head), the tile fastest
  const int b = blockIdx.y;
  const int pos = a.s.len[b], row = a.s.row[b];
  const int hs = unit / a.tiles, ti = unit - hs * a.tiles;
  const bool values = hs & 1;
  const int h = hs >> 1;
  const int tile = pos / kTile + ti, first = tile * kTile - pos;  // new position of the tile's first
  if (h >= a.p.heads || first >= a.len) return;                   // (a whole wave; no barrier follows)
  const bool full = first >= 0 && first + kTile <= a.len;
  const View &v = values ? a.v : a.k;
  const int piece = lane % PPR, sub = lane / PPR;
  const T *src = static_cast<const T *>(v.data) + b * v.s0 + h * v.s1 + 8 * piece;
  u32x4 raw[W][QW];
  int at[W];  // the new position of each load's row (not one: the nearest, in bounds)
#pragma unroll
  for (int w = 0; w < W; ++w) {
    at[w] = min(max(first + KPI * w + sub, 0), a.len - 1);
#pragma unroll
    for (int i = 0; i < QW; ++i) raw[w][i] = reinterpret_cast<const u32x4 *>(src + at[w] * v.s2)[i];
  }
  char *tp = tile4(a.p, row, tile, h);
  char *to = tp + (values ? 16 * D : 0);
  char *sto = tp + (values ? 34 : 32) * D;
  if (a.cos && !values) {
    // the angles' loads all before their first use (an empty statement holds them there)
    constexpr int STEP = sizeof(T) == 2 ? W : G;  // rows at a time
#pragma unroll
    for (int w0 = 0; w0 < W; w0 += STEP) {
      using Angles = std::conditional_t<sizeof(T) == 2, u32x2, u32x4>;
      Angles cw[STEP], sw[STEP];
#pragma unroll
      for (int j = 0; j < STEP; ++j) {
        const int64_t e = (static_cast<int64_t>(pos) + at[w0 + j]) * (D / 2) + 4 * piece;
        cw[j] = *reinterpret_cast<const Angles *>(static_cast<const T *>(a.cos) + e);
        sw[j] = *reinterpret_cast<const Angles *>(static_cast<const T *>(a.sin) + e);
      }
#pragma unroll
      for (int j = 0; j < STEP; ++j) asm volatile("" : "+v"(cw[j]), "+v"(sw[j]));
#pragma unroll
      for (int j = 0; j < STEP; ++j) {
        u32x4(&x)[QW] = raw[w0 + j];
        const T *cs = reinterpret_cast<const T *>(&cw[j]), *sn = reinterpret_cast<const T *>(&sw[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 2) {
            x[0][i] = rotate_word<T>(x[0][i], cs[i], sn[i], false);
          } else {
            const uint32_t u0 = x[i >> 1][2 * (i & 1)], u1 = x[i >> 1][2 * (i & 1) + 1];
            T x0 = __builtin_bit_cast(T, u0), x1 = __builtin_bit_cast(T, u1);
            rotate_pair(x0, x1, cs[i], sn[i], false);
            x[i >> 1][2 * (i & 1)] = __builtin_bit_cast(uint32_t, x0);
            x[i >> 1][2 * (i & 1) + 1] = __builtin_bit_cast(uint32_t, x1);
          }
        }
      }
    }
  }
  char *mine = lds[wv];
  uint16_t *scales = reinterpret_cast<uint16_t *>(mine + 16 * D);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float x[8];
#pragma unroll
    for (int i = 0; i < QW; ++i) {
      const T *e = reinterpret_cast<const T *>(&raw[w][i]);
#pragma unroll
      for (int j = 0; j < 8 / QW; ++j) x[i * (8 / QW) + j] = static_cast<float>(e[j]);
    }
    const float s = scale_of<T>(quad_umax(most_of<T>(raw[w])));
    const int key = KPI * w + sub;
    *reinterpret_cast<uint32_t *>(mine + word4<G>((key >> 4) * G + (piece >> 2), 16 * (piece & 3) + (key & 15))) =
        codes_of<T>(x, s == s ? s : 1.f);
    if ((piece & 3) == 0)
      scales[scale4<G>(key, piece >> 2)] = static_cast<uint16_t>(__builtin_bit_cast(uint32_t, s) >> 16);
  }
  wait_lgkm0();  // (own wave's writes)
  __builtin_amdgcn_sched_barrier(0);
  uint32_t word[W];
  load_words<G>(mine, lane, word);
  if (full) {
    if (lane < 4 * G) reinterpret_cast<u32x4 *>(sto)[lane] = reinterpret_cast<const u32x4 *>(scales)[lane];
  } else {
#pragma unroll
    for (int e0 = 0; e0 < 32 * G; e0 += 64) {
      const int e = e0 + lane, t = first + 16 * ((e >> 2) & 1) + 4 * (e / (8 * G)) + (e & 3);
      if (e < 32 * G && t >= 0 && t < a.len) reinterpret_cast<uint16_t *>(sto)[e] = scales[e];
    }
  }
  if (!values) {
    if (full) {
      store_words<G>(to, lane, word);
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int t = first + 16 * (w / G) + c;
        if (t >= 0 && t < a.len) *reinterpret_cast<uint32_t *>(to + word4<G>(w, lane)) = word[w];
      }
    }
    return;
  }
  const Transpose tr(lane);
  wait_lgkm0();  // (read before the next writes)
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int ks = 0; ks < G; ++ks) {
    uint32_t x = word[ks], y = word[G + ks];
    tr.to_values(x, y);
    *reinterpret_cast<uint32_t *>(mine + value_at<G>(c, g, ks, 0)) = x;
    *reinterpret_cast<uint32_t *>(mine + value_at<G>(c, g, ks, 1)) = y;
  }
  wait_lgkm0();  // (own wave's writes)
  __builtin_amdgcn_sched_barrier(0);
  load_words<G>(mine, lane, word);
  if (full) {
    store_words<G>(to, lane, word);
    return;
  }
  uint32_t keep = 0;  // codes of positions that are not new
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int t = first + 16 * (j >> 2) + 4 * g + (j & 3);
    if (t < 0 || t >= a.len) keep |= 0xFu << (4 * j);
  }
  if (keep != 0xFFFFFFFFu)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      uint32_t *old = reinterpret_cast<uint32_t *>(to + word4<G>(w, lane));
      *old = (*old & keep) | (word[w] & ~keep);
    }
}

struct ReadArgs {
  RowArgs r;
  int32_t first[kSeqs];  // the first position read
};

// Eight values of T from eight codes and their scale.
template <typename T>
__device__ __forceinline__ void store8(T *p, uint32_t w, float s, bool live) {
  f32x2 y[4];
  y[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
  y[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
  y[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
  y[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i][0] = live ? y[i][0] * s : 0.f;
    y[i][1] = live ? y[i][1] * s : 0.f;
  }
  if constexpr (sizeof(T) == 2) {
    __builtin_nontemporal_store(u32x4{pack2<T>(y[0][0], y[0][1]), pack2<T>(y[1][0], y[1][1]),
                                      pack2<T>(y[2][0], y[2][1]), pack2<T>(y[3][0], y[3][1])},
                                reinterpret_cast<u32x4 *>(p));
  } else {
    __builtin_nontemporal_store(f32x4{y[0][0], y[0][1], y[1][0], y[1][1]}, reinterpret_cast<f32x4 *>(p));
    __builtin_nontemporal_store(f32x4{y[2][0], y[2][1], y[3][0], y[3][1]}, reinterpret_cast<f32x4 *>(p) + 1);
  }
}

// The values of positions first .. first + len - 1 of every sequence into k, v
// [n, heads, len, D], zero past its length.  One wave a tile, head and side; the words
// go the append's way back, so that a store takes whole rows.  Bound by memory, most of
// it what is written, which nothing here reads again (stored past the caches): 4 x 8
// heads x 8192 positions of D128 in bf16, 172 MB, 27 us, 6.4 TB/s; 16 x 8 heads x 4001,
// 337 MB, 51 us, 6.6 TB/s (64 with ordinary stores, 82 with the operand order's 64-byte
// pieces of rows).
template <typename T, int G>
__global__ __launch_bounds__(NT) void read_kernel(ReadArgs ra) {
  constexpr int D = 32 * G, W = 2 * G;
  constexpr int PPR = D / 8, KPI = 64 / PPR;  // pieces a row, rows a store
  const RowArgs &a = ra.r;
  __shared__ __attribute__((aligned(16))) char lds[NW][16 * D];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x * NW + wv;
  const int b = blockIdx.y;
  const int hs = unit / a.tiles, ti = unit - hs * a.tiles;
  const bool values = hs & 1;
  const int h = hs >> 1;
  const int pos = ra.first[b], n = a.s.len[b];
  const int tile = pos / kTile + ti, first = tile * kTile - pos;  // output row of the tile's first
  if (h >= a.p.heads || first >= a.len) return;                   // (a whole wave; no barrier follows)
  const View &v = values ? a.v : a.k;
  T *out = static_cast<T *>(const_cast<void *>(v.data)) + b * v.s0 + h * v.s1;
  const int piece = lane % PPR, sub = lane / PPR;
  const bool held = tile * kTile < n;  // (a tile past the length may have no page)
  uint32_t word[W] = {};
  float sc[W] = {};
  if (held) {
    const char *base = tile4(a.p, a.s.row[b], tile, h);
    load_words<G>(base + (values ? 16 * D : 0), lane, word);
    const uint16_t *sfrom = reinterpret_cast<const uint16_t *>(base + (values ? 34 : 32) * D);
#pragma unroll
    for (int w = 0; w < W; ++w) sc[w] = from_bf16(sfrom[scale4<G>(KPI * w + sub, piece >> 2)]);
    char *mine = lds[wv];
    if (values) {  // to keys' words
      store_words<G>(mine, lane, word);
      wait_lgkm0();  // (own wave's writes)
      __builtin_amdgcn_sched_barrier(0);
      const Transpose tr(lane);
#pragma unroll
      for (int ks = 0; ks < G; ++ks) {
        word[ks] = *reinterpret_cast<const uint32_t *>(mine + value_at<G>(c, g, ks, 0));
        word[G + ks] = *reinterpret_cast<const uint32_t *>(mine + value_at<G>(c, g, ks, 1));
        tr.to_keys(word[ks], word[G + ks]);
      }
      wait_lgkm0();  // (read before the next writes)
      __builtin_amdgcn_sched_barrier(0);
    }
    store_words<G>(mine, lane, word);
    wait_lgkm0();  // (own wave's writes)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int key = KPI * w + sub;
      word[w] = *reinterpret_cast<const uint32_t *>(
          mine + word4<G>((key >> 4) * G + (piece >> 2), 16 * (piece & 3) + (key & 15)));
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int key = KPI * w + sub, t = first + key;
    if (t < 0 || t >= a.len) continue;
    store8<T>(out + static_cast<int64_t>(t) * v.s2 + 8 * piece, word[w], sc[w], tile * kTile + key < n);
  }
}

struct ApplyArgs {
  const char *from;
  char *to;
  int64_t page_bytes;
  int32_t *table;
  int32_t moves, sets;
  int32_t src[kMoves], dst[kMoves], at[kMoves], value[kMoves];
};

// Page copies, blockIdx.y's share of each: 16 bytes a lane, four loads in flight.  A
// launch of 168 pages of 73,728 bytes takes 7.2 us (3.3 TB/s), one of a few pages the
// launch's own 3; what a call has to copy is shorter than a second kernel for the table.
// The row of blocks past them writes table entries (whose pages the stream's next
// kernel reads: none here does).
__global__ __launch_bounds__(NT) void apply_kernel(ApplyArgs a) {
  const int move = blockIdx.y;
  if (move == a.moves) {
    const int i = blockIdx.x * NT + threadIdx.x;
    if (i < a.sets) a.table[a.at[i]] = a.value[i];
    return;
  }
  const u32x4 *from = reinterpret_cast<const u32x4 *>(a.from + a.src[move] * a.page_bytes);
  u32x4 *to = reinterpret_cast<u32x4 *>(a.to + a.dst[move] * a.page_bytes);
  const int64_t n = a.page_bytes / 16;
  constexpr int U = 4;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * NT * U; i0 < n; i0 += static_cast<int64_t>(gridDim.x) * NT * U) {
    u32x4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * NT + threadIdx.x;
      r[u] = __builtin_nontemporal_load(from + (i < n ? i : n - 1));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * NT + threadIdx.x;
      if (i < n) __builtin_nontemporal_store(r[u], to + i);
    }
  }
}

// f(T, G) for the cache's dtype and head dim (both checked by the caller).
template <typename F>
void by_type(int dtype, int dim, F &&f) {
  auto dims = [&](auto t) {
    if (dim == 32) f(t, std::integral_constant<int, 1>{});
    else if (dim == 64) f(t, std::integral_constant<int, 2>{});
    else if (dim == 128) f(t, std::integral_constant<int, 4>{});
    else f(t, std::integral_constant<int, 8>{});
  };
  if (dtype == TSATTN_F32) dims(float{});
  else if (dtype == TSATTN_F16) dims(f16{});
  else dims(bf16{});
}

}  // namespace

hipError_t launch_pages4_append(const Pages4 &p, int dtype, int n, int len, View k, View v, const Seqs &s,
                                const void *cos, const void *sin, hipStream_t st) {
  // a sequence's len new positions touch at most (len + 30) / 32 + 1 tiles
  const RowArgs a{p, s, k, v, cos, sin, len, (len + kTile - 2) / kTile + 1};
  const int64_t units = static_cast<int64_t>(a.tiles) * p.heads * 2;
  const dim3 grid(static_cast<unsigned>((units + NW - 1) / NW), n);
  Probe pr_("pages4_append", st);
  by_type(dtype, p.dim, [&](auto t, auto g) {
    append_kernel<decltype(t), decltype(g)::value><<<grid, dim3(NT), 0, st>>>(a);
  });
  return hipGetLastError();
}

hipError_t launch_pages4_read(const Pages4 &p, int dtype, int n, int len, View k, View v, const Seqs &s,
                              const int32_t *first, hipStream_t st) {
  ReadArgs a{RowArgs{p, s, k, v, nullptr, nullptr, len, (len + kTile - 2) / kTile + 1}, {}};
  for (int i = 0; i < n; ++i) a.first[i] = first[i];
  const int64_t units = static_cast<int64_t>(a.r.tiles) * p.heads * 2;
  const dim3 grid(static_cast<unsigned>((units + NW - 1) / NW), n);
  Probe pr_("pages4_read", st);
  by_type(dtype, p.dim, [&](auto t, auto g) {
    read_kernel<decltype(t), decltype(g)::value><<<grid, dim3(NT), 0, st>>>(a);
  });
  return hipGetLastError();
}

hipError_t launch_pages4_apply(const char *from, char *to, int64_t page_bytes, int moves, const int32_t *src,
                               const int32_t *dst, int32_t *table, int sets, const int32_t *at,
                               const int32_t *value, hipStream_t st) {
  const int64_t whole = moves ? (page_bytes / 16 + NT * 4 - 1) / (NT * 4) : 1;
  const unsigned least = (kMoves + NT - 1) / NT, most = 64;  // (the entries' blocks; enough for a page)
  const unsigned bx = whole < least ? least : whole < most ? static_cast<unsigned>(whole) : most;
  Probe pr_("pages4_apply", st);
  for (int i0 = 0; i0 < moves || i0 < sets; i0 += kMoves) {
    ApplyArgs a{from, to, page_bytes, table, 0, 0, {}, {}, {}, {}};
    for (; a.moves < kMoves && i0 + a.moves < moves; ++a.moves)
      a.src[a.moves] = src[i0 + a.moves], a.dst[a.moves] = dst[i0 + a.moves];
    for (; a.sets < kMoves && i0 + a.sets < sets; ++a.sets)
      a.at[a.sets] = at[i0 + a.sets], a.value[a.sets] = value[i0 + a.sets];
    apply_kernel<<<dim3(bx, a.moves + (a.sets ? 1 : 0)), dim3(NT), 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tsattn
