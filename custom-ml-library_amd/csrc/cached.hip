// Attention of a few new tokens over a key/value cache that they do not all see alike: a
// sliding window with sinks, or a tree of drafted tokens.  f16, bf16, int8 (codes with a
// scale a row) and f32 caches.
//
// Token t's position is P + its depth, P the positions in front of the new ones (a chain:
// depth t).  It sees key j < P where j < sinks or j > position - window, and of the new
// keys those up to its own (chain) or its ancestors' and its own (tree, a bit each).  Which
// of 32 keys a row sees is one word, made of three comparisons and the tree's bits; only
// tiles at the window's border, the sinks' last and the new ones need it.
//
// The rows of a KV head (its query heads times the tokens) are the columns of S^T = K Q^T,
// 32 to a wave, so that the statistics of a row are a lane's own and P^T is the operand of
// O^T += V^T P^T as it comes.  Every wave works alone on tiles of its own through its own
// LDS ring and the waves' results are joined at the end, or, for many rows of many heads, 4
// waves of 32 rows share each tile (plan_cached).  The tiles that a window leaves lie in one
// run, which splits cut into equal parts, as many as fill the chip; a second kernel joins
// those.
//
// Bound by HBM for few rows (keys and values once), by the softmax beside the matrix
// instructions from about 100 rows a KV head on.
//
// P is rounded to the cache's type for the second product, as in the prefill kernel; f32
// keeps it.  Over int8 caches the codes are exact in 16 bits, keys' scales multiply the
// scores, values' scales P, which then may be small and so is rounded to bf16, for f16
// queries as the sum of two.
#include <type_traits>

#include "f32_tile.h"
#include "rope_math.h"

namespace tsattn {
namespace {

constexpr int BN = 32;  // keys per tile
constexpr float kTau = 8.f;

struct CachedArgs {
  int B, Hkv, rep, T, n, R;  // R = rep T rows a KV head
  View q, k, v, o, ks, vs;
  const uint32_t *words;
  const int32_t *depth;
  int tree_rows, W;
  int window, sinks;
  int ns, gap, run;  // the tiles in use: ns of the sinks, then those `gap` further on
  int splits, groups;
  float sl;  // scale * log2(e)
  RopeDesc rope;
  float *ws;  // partial O [splits][B Hkv R][D], then [splits][B Hkv R][2] (max, sum)
};

template <typename T, int D>
constexpr int kPair = 2 * BN * D * (std::is_same_v<T, float> ? 4 : 2);  // bytes of a K and a V tile, in T
// Waves of a workgroup, WR of them sharing each tile.  A wave of its own (WR 1) has room
// for one K and one V tile of 16 bits, so that 8 waves of 128 channels share a CU: with
// room for more, 4 waves and 3 or 4 of a wave's tiles in flight, the step that plan_cached
// names took the same time.
template <typename T, int D, int WR>
constexpr int kWaves = WR > 1 ? WR : (kPair<T, D> <= 16384 ? 4 : 2);
// Waves a SIMD that the registers must leave room for.
template <typename T, int D>
constexpr int kTwo = kPair<T, D> <= 16384 ? 2 : 1;
// Ring stages of a K and a V tile: of 4 waves four, of one wave one, or two of codes, half
// as large.
template <bool Q8, int WR>
constexpr int kStages = WR > 1 ? 4 : Q8 ? 2 : 1;

__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// Eight int8 codes as eight values of T (exact).  In f16, 1024 + (code + 128) is a code
// with its sign bit turned under the exponent byte 0x64, two to a permutation and a sum.
template <typename T>
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
  u32x4 y;
  if constexpr (std::is_same_v<T, f16>) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = (i < 2 ? lo : hi) ^ 0x80808080u;
      const uint32_t two = __builtin_amdgcn_perm(0x64646464u, u, i & 1 ? 0x04030402u : 0x04010400u);
      y[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, two) + h2{-1152, -1152});
    }
    return y;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? lo : hi) >> (16 * (i & 1));
    y[i] = pack2<T>(static_cast<float>(static_cast<int8_t>(w & 0xFFu)),
                    static_cast<float>(static_cast<int8_t>((w >> 8) & 0xFFu)));
  }
  return y;
}

// Code n of a lane's 8 bytes.
__device__ __forceinline__ float code(u32x2 x, int n) {
  return static_cast<float>(static_cast<int8_t>((x[n >> 2] >> (8 * (n & 3))) & 0xFFu));
}

// 16-bit K / V tiles in LDS, 32 rows of D, row-major, 16-byte chunk k of row r at k ^
// sw(r).  One DMA instruction fetches whole rows.  16 rows' same chunk, and 4 rows' 4
// chunks beside each other (the transposing reads), lie in different banks.
template <typename T, int D>
struct RowTile {
  static constexpr int RPB = 1024 / (2 * D);  // rows a DMA block
  __device__ __forceinline__ static constexpr int sw(int r) {
    return D >= 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : D == 64 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : (r >> 2) & 3;
  }
  // of the block's first row: what lane l fetches for its 16 bytes at 16 l of block n
  __device__ __forceinline__ static uint32_t dma_off(int n, int lane, uint32_t stride) {
    const int rr = lane / (D / 8), k = lane % (D / 8);
    return static_cast<uint32_t>(rr) * stride + static_cast<uint32_t>((k ^ sw(n * RPB + rr)) << 4);
  }
  int krow, kchunk, vrow, vlo, vhi;
  __device__ __forceinline__ explicit RowTile(int lane) {
    const int c = lane & 31, h = lane >> 5, i = lane & 15, sel = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    const int r = 4 * h + (i >> 2);
    krow = c * 2 * D, kchunk = (h ^ sw(c)) << 4;
    vrow = r * 2 * D + (i & 1) * 8, vlo = (sel ^ sw(r)) << 4, vhi = (sel ^ sw(r + 8)) << 4;
  }
  // row c, channels 16 i + 8 h .. + 7
  __device__ __forceinline__ u32x4 rows(const char *tile, int i) const {
    return ld16(tile + krow + (kchunk ^ (i << 5)));
  }
  // channel 32 dt + c at rows 16 ks + 4 h .. + 3 and 8 further on
  __device__ __forceinline__ u32x4 cols(const char *tile, int ks, int dt) const {
    const char *t = tile + vrow + ks * 32 * D;
    const u32x2 a = ds_read_tr<T>(reinterpret_cast<const T *>(t + (vlo ^ (dt << 6))));
    const u32x2 b = ds_read_tr<T>(reinterpret_cast<const T *>(t + 16 * D + (vhi ^ (dt << 6))));
    return u32x4{a[0], a[1], b[0], b[1]};
  }
};

// Tiles of int8 codes, 32 rows of D bytes, the 16-byte chunk k of row r at k ^ sw(r): 16
// rows' same chunk lie in different banks.  They are widened on the way to the matrix
// instructions (through registers into 16-bit tiles in LDS instead, a window's step over 32
// sequences' 4096 keys of 8 heads of 128 took 148 us, so 54, 5 TB/s; of 256 channels, whose
// registers spilled, 16 sequences 627 and 60), which fixes the order of a lane's channels
// in both products:
//   scores: step 2 j + e contracts channels 32 j + 16 h + 8 e .. + 7, a chunk for two steps;
//   values: row c of block dt of O^T is channel D / 32 c + dt, so that a lane's D / 32
//   neighbouring bytes of a key serve one block each and nothing is transposed.
template <int D>
struct CodeTile {
  static constexpr int RPB = 1024 / D, CPR = D / 16, PDT = D / 32;
  __device__ __forceinline__ static constexpr int sw(int r) { return r * CPR / 16 & (CPR - 1); }
  __device__ __forceinline__ static uint32_t dma_off(int n, int lane, uint32_t stride) {
    const int rr = lane / CPR, k = lane % CPR;
    return static_cast<uint32_t>(rr) * stride + static_cast<uint32_t>((k ^ sw(n * RPB + rr)) << 4);
  }
  int krow, kchunk, vbyte, h;
  __device__ __forceinline__ explicit CodeTile(int lane) {
    const int c = lane & 31;
    h = lane >> 5;
    krow = c * D, kchunk = (h ^ sw(c)) << 4;
    vbyte = (c * PDT) ^ (sw(4 * h) << 4);
  }
  // row c, channels 32 j + 16 h .. + 15
  __device__ __forceinline__ u32x4 rows(const char *tile, int j) const { return ld16(tile + krow + (kchunk ^ (j << 5))); }
  // key 16 ks + 8 a + 4 h + b, channels PDT c .. + PDT - 1
  __device__ __forceinline__ u32x2 key(const char *tile, int ks, int a, int b) const {
    const char *at = tile + (16 * ks + 8 * a + 4 * h + b) * D + (vbyte ^ (sw(8 * a + b) << 4));
    if constexpr (PDT == 8) return *reinterpret_cast<const u32x2 *>(at);
    else if constexpr (PDT == 4) return u32x2{*reinterpret_cast<const uint32_t *>(at), 0u};
    else if constexpr (PDT == 2) return u32x2{*reinterpret_cast<const uint16_t *>(at), 0u};
    else return u32x2{*reinterpret_cast<const uint8_t *>(at), 0u};
  }
};

// Lane l's 4 bytes at voff + soff go to LDS at lds + 4 l.
__device__ __forceinline__ void dma4(u32x4 desc, uint32_t lds, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(desc),
                 "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory", "m0");
}

template <typename T, int D, bool Q8, int WR, bool NT>
__global__ __launch_bounds__((64 * kWaves<T, D, WR>), (kTwo<T, D>)) void cached_kernel(CachedArgs a) {
  constexpr bool F32 = std::is_same_v<T, float>;
  static_assert(!F32 || (!Q8 && D <= 128), "fp32 caches are not quantised, of up to 128 channels");
  static_assert(WR == 1 || (!F32 && !Q8), "waves share tiles of 16 bits");
  using PT = std::conditional_t<Q8, bf16, T>;  // the value tiles
  constexpr int NP = Q8 && std::is_same_v<T, f16> ? 2 : 1;  // parts of P
  constexpr int NWV = kWaves<T, D, WR>, WK = NWV / WR, NS = kStages<Q8, WR>;
  constexpr int PAIR = Q8 ? kPair<T, D> / 2 : kPair<T, D>, TILE = PAIR / 2;
  constexpr int BLK = TILE / 1024;        // 1 KiB DMA blocks a tile
  constexpr int LK = BLK + (Q8 ? 2 : 0), LV = BLK;  // loads of a K tile (and both tiles' scales), a V tile
  constexpr int LPT = (LK + LV) / WR;               // loads a wave issues for a pair (WR > 1)
  constexpr int PDT = D / 32;
  // the stages, then (codes) one place more for 64 floats of K's and 64 of V's scales, half
  // of each in use: a tile's are read after its K's place is loaded again
  constexpr int RING = NS * PAIR + (Q8 ? (NS + 1) * 512 : 0);
  constexpr int MERGE = WK > 1 ? NWV * 32 * (D + 2) * 4 : 0;
  constexpr int LDS_B = WK * RING > MERGE ? WK * RING : MERGE;
  static_assert((LK + LV) % WR == 0 && (WR > 1 ? LPT : NS * (LK + LV)) < 64, "loads in flight that a wait can count");
  __shared__ __attribute__((aligned(1024))) char lds[LDS_B];

  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = WR > 1 ? w : 0, wk = WR > 1 ? 0 : w;
  // row groups of the same keys follow each other, on one XCD
  const int bhs = a.B * a.Hkv;
  const int logical = xcd_remap(blockIdx.x, bhs * a.splits * a.groups);
  const int rg = logical % a.groups, part = logical / a.groups % a.splits, bh = logical / (a.groups * a.splits);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int t0 = static_cast<int>(static_cast<int64_t>(a.run) * part / a.splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(a.run) * (part + 1) / a.splits);
  const int mine = t1 - t0 > wk ? (t1 - t0 - wk - 1) / WK + 1 : 0;  // this wave's tiles
  auto key0 = [&](int i) __attribute__((always_inline)) {  // the first key of its tile i
    const int j = t0 + wk + WK * i;
    return BN * (j < a.ns ? j : j + a.gap);
  };

  // this lane's row
  const int row = (rg * WR + wr) * 32 + c;
  const bool live = row < a.R;
  const int rr = live ? row / a.T : 0, t = live ? row - rr * a.T : 0;
  const int64_t tree = static_cast<int64_t>(a.tree_rows > 1 ? b : 0) * a.T + t;
  const int P = a.n - a.T;
  const int pos = P + (a.words ? a.depth[tree] : t);
  const uint32_t *words = a.words ? a.words + tree * a.W : nullptr;
  const int low = a.window ? pos - a.window + 1 : 0;
  // Which of the 32 keys from kv0 on the row sees.
  auto visible = [&](int kv0) {
    uint32_t seen = low_bits(a.sinks - kv0) | ~low_bits(low - kv0);
    const int off = kv0 - P;
    if (off > -BN) {
      uint32_t x;
      if (!words) {
        x = low_bits(t + 1 - off);
      } else if (off < 0) {
        x = (words[0] << -off) | low_bits(-off);
      } else {
        const int i = off >> 5, sh = off & 31;
        x = i < a.W ? words[i] >> sh : 0u;
        if (sh && i + 1 < a.W) x |= words[i + 1] << (32 - sh);
      }
      seen &= x;
    }
    return seen;
  };
  // keys below `border` are hidden from some row
  const int border = a.window ? a.n - a.window : 0;

  // Q rows as B operands: 16-bit, channels 16 ks + 8 h .. + 7 (over codes in CodeTile's
  // order); f32, the half h of the row
  constexpr int NQ = F32 ? D / 8 : D / 16;  // 16-byte pieces a lane holds
  u32x4 qf[NQ];
  {
    const T *qp = static_cast<const T *>(a.q.data) + b * a.q.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.q.s1 +
                  static_cast<int64_t>(t) * a.q.s2 + (F32 ? h * (D / 2) : Q8 ? 16 * h : 8 * h);
    auto channel = [](int i) { return F32 ? 4 * i : Q8 ? 32 * (i >> 1) + 8 * (i & 1) : 16 * i; };
#pragma unroll
    for (int i = 0; i < NQ; ++i) qf[i] = ld16(qp + channel(i));
    if (a.rope.R > 0) {
      if constexpr (F32) {
        const float *cs = static_cast<const float *>(a.rope.cos) + static_cast<int64_t>(pos) * (D / 2) + h * (D / 4);
        const float *sn = static_cast<const float *>(a.rope.sin) + static_cast<int64_t>(pos) * (D / 2) + h * (D / 4);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t b0 = qf[i][2 * e], b1 = qf[i][2 * e + 1];
            float x0 = __builtin_bit_cast(float, b0), x1 = __builtin_bit_cast(float, b1);
            rotate_pair(x0, x1, cs[2 * i + e], sn[2 * i + e], false);
            qf[i][2 * e] = __builtin_bit_cast(uint32_t, x0), qf[i][2 * e + 1] = __builtin_bit_cast(uint32_t, x1);
          }
      } else {
        int64_t at[NQ];
        int p0[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) at[i] = pos, p0[i] = (channel(i) + (Q8 ? 16 : 8) * h) / 2;
        rotate_chunks<T, NQ>(qf, a.rope, at, p0, false);
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if (!live) qf[i] = u32x4{0, 0, 0, 0};
      asm volatile("" : "+v"(qf[i]));  // loaded before the DMA stream starts
    }
  }

  f32x16 oacc[PDT];
#pragma unroll
  for (int dt = 0; dt < PDT; ++dt) oacc[dt] = f32x16{};
  float m = -INFINITY, l = 0.f, thr = -INFINITY, nbase = 0.f;
  const float sl = a.sl, inv_sl = 1.f / sl;
  char *ring = lds + wk * RING;
  const uint32_t ring0 = lds_addr(lds) + wk * RING;

  using Tile = std::conditional_t<F32, FTile<D>, std::conditional_t<Q8, CodeTile<D>, RowTile<std::conditional_t<F32, bf16, T>, D>>>;
  const std::conditional_t<F32, RowTile<bf16, D>, Tile> rd(lane);  // (FTile's reads keep no state)
  // S^T of a K tile: element i is key crow(i, h)
  auto scores = [&](const char *kt) __attribute__((always_inline)) {
    f32x16 s = f32x16{};
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const float4 x = FTile<D>::chunk(kt, c, h * NQ + i);
        const uint32_t q0 = qf[i][0], q1 = qf[i][1], q2 = qf[i][2], q3 = qf[i][3];
        s = mfma32f(x.x, __builtin_bit_cast(float, q0), s);
        s = mfma32f(x.y, __builtin_bit_cast(float, q1), s);
        s = mfma32f(x.z, __builtin_bit_cast(float, q2), s);
        s = mfma32f(x.w, __builtin_bit_cast(float, q3), s);
      }
    } else if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < NQ / 2; ++j) {
        const u32x4 x = rd.rows(kt, j);
        s = mfma32<T>(widen<T>(x[0], x[1]), qf[2 * j], s);
        s = mfma32<T>(widen<T>(x[2], x[3]), qf[2 * j + 1], s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NQ; ++i) s = mfma32<T>(rd.rows(kt, i), qf[i], s);
    }
    return s;
  };
  float p[16];                  // P of the tile (f32 caches)
  u32x4 pb[NP][F32 ? 1 : 2];    // or its packed parts
  // The softmax of the tile from kv0 on; scales: its keys' (Q8), then its values'.
  auto softmax = [&](f32x16 s, int kv0, const float *scales) __attribute__((always_inline)) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = s[i];
    if constexpr (Q8) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 f = *reinterpret_cast<const float4 *>(scales + 8 * g + 4 * h);
        x[4 * g] *= f.x, x[4 * g + 1] *= f.y, x[4 * g + 2] *= f.z, x[4 * g + 3] *= f.w;
      }
    }
    if (kv0 + BN > P || (kv0 < border && kv0 + BN > a.sinks)) {
      const uint32_t seen = visible(kv0) >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = (seen >> (8 * (i >> 2) + (i & 3))) & 1u ? x[i] : -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    const float mxr = half_swap_max3(mx);
    if (__ballot(mxr > thr) != 0ull) {
      const float m_new = fmaxf(m, mxr * sl);
      const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m - m_new);
      m = m_new;
      thr = (m + kTau) * inv_sl;
      nbase = m == -INFINITY ? 0.f : -m;
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < PDT; ++dt) oacc[dt] *= corr;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = fast_exp2(fmaf(x[i], sl, nbase));
      l += p[i];
    }
    if constexpr (Q8) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 f = *reinterpret_cast<const float4 *>(scales + 64 + 8 * g + 4 * h);
        p[4 * g] *= f.x, p[4 * g + 1] *= f.y, p[4 * g + 2] *= f.z, p[4 * g + 3] *= f.w;
      }
    }
    if constexpr (!F32) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const uint32_t hi = pack2<PT>(p[i], p[i + 1]);
        pb[0][i >> 3][(i & 7) >> 1] = hi;
        if constexpr (NP > 1) {  // (bf16) what the first part leaves
          const uint32_t h0 = hi << 16, h1 = hi & 0xFFFF0000u;
          pb[1][i >> 3][(i & 7) >> 1] =
              pack2<PT>(p[i] - __builtin_bit_cast(float, h0), p[i + 1] - __builtin_bit_cast(float, h1));
        }
      }
    }
  };
  auto values = [&](const char *vt) __attribute__((always_inline)) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int dt = 0; dt < PDT; ++dt)
          oacc[dt] = mfma32f(FTile<D>::elem(vt, 8 * (i >> 2) + 4 * h + (i & 3), 32 * dt + c), p[i], oacc[dt]);
    } else if constexpr (Q8) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x2 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = rd.key(vt, ks, j >> 2, j & 3);
#pragma unroll
        for (int dt = 0; dt < PDT; ++dt) {
          u32x4 f;
#pragma unroll
          for (int j = 0; j < 8; j += 2) f[j >> 1] = pack2<PT>(code(x[j], dt), code(x[j + 1], dt));
#pragma unroll
          for (int n = 0; n < NP; ++n) oacc[dt] = mfma32<PT>(f, pb[n][ks], oacc[dt]);
        }
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int dt = 0; dt < PDT; ++dt) {
          const u32x4 f = rd.cols(vt, ks, dt);
#pragma unroll
          for (int n = 0; n < NP; ++n) oacc[dt] = mfma32<PT>(f, pb[n][ks], oacc[dt]);
        }
    }
  };

  using KT = std::conditional_t<Q8, int8_t, T>;
  const uint32_t ks_b = static_cast<uint32_t>(a.k.s2) * sizeof(KT), vs_b = static_cast<uint32_t>(a.v.s2) * sizeof(KT);
  const KT *kbase = static_cast<const KT *>(a.k.data) + b * a.k.s0 + hk * a.k.s1;
  const KT *vbase = static_cast<const KT *>(a.v.data) + b * a.v.s0 + hk * a.v.s1;
  // Keys past the cache's end, and tiles past the wave's last, read as zeros.
  const u32x4 kdesc = make_desc(kbase, static_cast<uint32_t>(a.n) * ks_b);
  const u32x4 vdesc = make_desc(vbase, static_cast<uint32_t>(a.n) * vs_b);
  u32x4 ksdesc{}, vsdesc{};
  uint32_t kss_b = 0, vss_b = 0;
  if constexpr (Q8) {
    kss_b = static_cast<uint32_t>(a.ks.s2) * 4, vss_b = static_cast<uint32_t>(a.vs.s2) * 4;
    ksdesc = make_desc(static_cast<const float *>(a.ks.data) + b * a.ks.s0 + hk * a.ks.s1, static_cast<uint32_t>(a.n) * kss_b);
    vsdesc = make_desc(static_cast<const float *>(a.vs.data) + b * a.vs.s0 + hk * a.vs.s1, static_cast<uint32_t>(a.n) * vss_b);
  }
  auto first_row = [&](int i, uint32_t stride) __attribute__((always_inline)) {
    return i < mine ? static_cast<uint32_t>(key0(i)) * stride : 0x80000000u;
  };
  // load n of tile i: K's blocks, the scales, V's blocks
  struct At {
    uint32_t st, sc, k, v, ks, vs;
  };
  auto place = [&](int i) __attribute__((always_inline)) {
    At t{ring0 + (i % NS) * PAIR, 0, first_row(i, ks_b), first_row(i, vs_b), 0, 0};
    if constexpr (Q8) t.sc = ring0 + NS * PAIR + (i % (NS + 1)) * 512, t.ks = first_row(i, kss_b), t.vs = first_row(i, vss_b);
    return t;
  };
  auto fetch = [&](u32x4 desc, uint32_t to, uint32_t off, uint32_t base) __attribute__((always_inline)) {
    if constexpr (NT) dma16_nt(desc, to, off, base);
    else dma16(desc, to, off, base);
  };
  auto load = [&](const At &t, int n) __attribute__((always_inline)) {
    if (n < BLK) {
      fetch(kdesc, t.st + n * 1024, Tile::dma_off(n, lane, ks_b), t.k + static_cast<uint32_t>(n * Tile::RPB) * ks_b);
    } else if (!Q8 || n >= LK) {
      const int at = n - LK;
      fetch(vdesc, t.st + TILE + at * 1024, Tile::dma_off(at, lane, vs_b), t.v + static_cast<uint32_t>(at * Tile::RPB) * vs_b);
    } else if (n == BLK) {  // (lanes 32 .. 63 fetch the same again)
      dma4(ksdesc, t.sc, static_cast<uint32_t>(lane & 31) * kss_b, t.ks);
    } else {
      dma4(vsdesc, t.sc + 256, static_cast<uint32_t>(lane & 31) * vss_b, t.vs);
    }
  };
  auto scales_of = [&](int i) __attribute__((always_inline)) {
    return reinterpret_cast<const float *>(ring + NS * PAIR + (i % (NS + 1)) * 512);
  };
  if constexpr (WR == 1) {
    // a tile's places are loaded again, NS tiles on, as soon as they are read
    auto issue = [&](int i, int from, int to) __attribute__((always_inline)) {
      const At t = place(i);
#pragma unroll
      for (int n = from; n < to; ++n) load(t, n);
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) issue(i, 0, LK + LV);
    for (int i = 0; i < mine; ++i) {
      const char *kt = ring + (i % NS) * PAIR;
      wait_vm_n<NS * LV + (NS - 1) * LK>();  // K of tile i; V and what follows in flight
      __builtin_amdgcn_sched_barrier(0);
      const f32x16 s = scores(kt);
      wait_lgkm0();  // read
      __builtin_amdgcn_sched_barrier(0);
      issue(i + NS, 0, LK);
      softmax(s, key0(i), scales_of(i));
      __builtin_amdgcn_sched_barrier(0);
      wait_vm_n<NS * LK + (NS - 1) * LV>();  // V of tile i
      __builtin_amdgcn_sched_barrier(0);
      values(kt + TILE);
      wait_lgkm0();
      __builtin_amdgcn_sched_barrier(0);
      issue(i + NS, LK, LK + LV);
    }
    wait_vm_n<0>();
  } else {
    // wave w issues loads w, w + WR, .. of a pair, three tiles ahead
    auto issue = [&](int i) __attribute__((always_inline)) {
      const At t = place(i);
#pragma unroll
      for (int u = 0; u < LPT; ++u) {
        const int n = w + WR * u;
        if (WR * u + WR <= BLK) __builtin_assume(n < BLK);  // (a K block whatever the wave: no branch)
        else if (WR * u >= LK) __builtin_assume(n >= LK);
        load(t, n);
      }
    };
    // O^T += V^T P^T of a tile and the next one's scores are one run of matrix
    // instructions, among which the exponentials issue; the ring's stages are unrolled,
    // so that LDS addresses are constants beside the lane's (63 tokens of 16 sequences
    // over 8000 keys, bf16: 170 us each tile by itself with three stages, 157 this way,
    // 150 unrolled; fragments read 3 steps ahead by hand, or a higher priority during
    // the matrix instructions: no change)
    issue(0);
    issue(1);
    issue(2);
    wait_vm_n<2 * LPT>();
    phase_barrier();
    f32x16 s = scores(ring);
    auto step = [&](int i, auto stage) __attribute__((always_inline)) {
      softmax(s, key0(i), scales_of(i));
      wait_vm_n<LPT>();  // this wave's loads of tile i + 1
      wait_lgkm0();
      phase_barrier();  // every wave's; and tile i - 1 is read
      issue(i + 3);
      s = scores(ring + (stage + 1) % NS * PAIR);
      values(ring + stage * PAIR + TILE);
    };
    for (int i = 0; i < mine; i += NS) {
      step(i, std::integral_constant<int, 0>{});
      if (i + 1 < mine) step(i + 1, std::integral_constant<int, 1>{});
      if (i + 2 < mine) step(i + 2, std::integral_constant<int, 2>{});
      if (i + 3 < mine) step(i + 3, std::integral_constant<int, 3>{});
    }
    wait_vm_n<0>();
  }

  // Lane holds O^T[row 8 g + 4 h + r of block dt][row c] in oacc[dt][4 g + r]: four
  // neighbouring channels are r = 0 .. 3 of a block, over codes (CodeTile) of D / 32 blocks
  // side by side.
  auto block_of = [](int q, int j) { return Q8 ? (4 * (q % PDT) + j) % PDT : q >> 2; };
  auto element = [](int q, int j) { return Q8 ? 4 * (q / PDT) + (4 * (q % PDT) + j) / PDT : 4 * (q & 3) + j; };
  auto channel4 = [&](int q) { return Q8 ? PDT * (8 * (q / PDT) + 4 * h) + 4 * (q % PDT) : 8 * q + 4 * h; };
  const int64_t rows = static_cast<int64_t>(bhs) * a.R, at = static_cast<int64_t>(bh) * a.R + row;
  float *po = a.ws + (part * rows + at) * D;
  float *ml = a.ws + a.splits * rows * D + 2 * (part * rows + at);
  T *out = static_cast<T *>(const_cast<void *>(a.o.data)) + b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
           static_cast<int64_t>(t) * a.o.s2;
  auto store = [&](int d, float4 x, float inv) __attribute__((always_inline)) {
    if (a.splits > 1) {
      *reinterpret_cast<float4 *>(po + d) = x;
    } else if constexpr (F32) {
      *reinterpret_cast<float4 *>(out + d) = float4{x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    } else {
      *reinterpret_cast<u32x2 *>(out + d) = u32x2{pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv)};
    }
  };
  float lt = xor32_sum(l);
  if constexpr (WK == 1) {
    if (!live) return;
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
#pragma unroll
    for (int q = 0; q < 4 * PDT; ++q)
      store(channel4(q),
            float4{oacc[block_of(q, 0)][element(q, 0)], oacc[block_of(q, 1)][element(q, 1)],
                   oacc[block_of(q, 2)][element(q, 2)], oacc[block_of(q, 3)][element(q, 3)]}, inv);
  } else {
    // the waves' results, joined in their order; wave w stores fours w, w + NWV, .. of channels
    __syncthreads();  // every ring is read
    float *cm = reinterpret_cast<float *>(lds), *cl = cm + NWV * 32, *co = cl + NWV * 32;
    if (h == 0) cm[w * 32 + c] = m, cl[w * 32 + c] = lt;
#pragma unroll
    for (int dt = 0; dt < PDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) co[((w * PDT + dt) * 16 + e) * 64 + lane] = oacc[dt][e];
    __syncthreads();
    m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NWV; ++v) m = fmaxf(m, cm[v * 32 + c]);
    float f[NWV];
    lt = 0.f;
#pragma unroll
    for (int v = 0; v < NWV; ++v) {
      const float mv = cm[v * 32 + c];
      f[v] = mv == -INFINITY ? 0.f : fast_exp2(mv - m);
      lt += cl[v * 32 + c] * f[v];
    }
    if (!live) return;
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
    for (int q = w; q < PDT * 4; q += NWV) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < NWV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[r] = fmaf(co[((v * PDT + block_of(q, r)) * 16 + element(q, r)) * 64 + lane], f[v], x[r]);
      store(channel4(q), float4{x[0], x[1], x[2], x[3]}, inv);
    }
    if (w) return;
  }
  if (a.splits > 1 && h == 0) ml[0] = m, ml[1] = lt;
}

// The splits' partial rows, joined in their order: D / 4 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void cached_merge_kernel(CachedArgs a) {
  constexpr int LPR = D / 4, RPB = 256 / LPR;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.R;
  const int q = threadIdx.x % LPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LPR;
  if (row >= rows) return;
  const float *ml = a.ws + a.splits * rows * D + 2 * row;
  float M = -INFINITY;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, ml[2 * s * rows]);
  float L = 0.f;
  float4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float mv = ml[2 * s * rows];
    const float f = mv == -INFINITY ? 0.f : fast_exp2(mv - M);
    L = fmaf(ml[2 * s * rows + 1], f, L);
    const float4 x = *reinterpret_cast<const float4 *>(a.ws + (s * rows + row) * D + 4 * q);
    o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int64_t bh = row / a.R, b = bh / a.Hkv;
  const int r = static_cast<int>(row - bh * a.R), hk = static_cast<int>(bh - b * a.Hkv);
  T *op = static_cast<T *>(const_cast<void *>(a.o.data)) + b * a.o.s0 +
          static_cast<int64_t>(hk * a.rep + r / a.T) * a.o.s1 + static_cast<int64_t>(r % a.T) * a.o.s2 + 4 * q;
  if constexpr (std::is_same_v<T, float>)
    *reinterpret_cast<float4 *>(op) = float4{o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  else
    *reinterpret_cast<u32x2 *>(op) = u32x2{pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv)};
}

// ---------------------------------------------------------------------------
// A tree's words and depths from its parents: a workgroup a tree, the ancestors found by
// doubling (each round a token takes over the ancestors of the furthest one it knows).
// ---------------------------------------------------------------------------
constexpr int kMostTokens = 256, kWords = kMostTokens / 32;

__global__ __launch_bounds__(kMostTokens) void draft_tree_kernel(int T, const int32_t *parents, uint32_t *words,
                                                                 int32_t *depth) {
  __shared__ uint32_t up[kMostTokens][kWords];
  __shared__ int jump[kMostTokens];
  const int t = threadIdx.x;
  uint32_t mine[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) up[t][i] = mine[i] = t >> 5 == i ? 1u << (t & 31) : 0u;
  const int parent = t < T ? parents[static_cast<int64_t>(blockIdx.x) * T + t] : -1;
  int to = parent >= 0 && parent < t ? parent : -1;
  jump[t] = to;
  __syncthreads();
  for (int far = 1; far < T; far <<= 1) {
    int next = -1;
    if (to >= 0) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) mine[i] |= up[to][i];
      next = jump[to];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWords; ++i) up[t][i] = mine[i];
    jump[t] = to = next;
    __syncthreads();
  }
  if (t >= T) return;
  const int W = (T + 31) / 32;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kWords; ++i) n += __popc(mine[i]);
  for (int i = 0; i < W; ++i) words[(static_cast<int64_t>(blockIdx.x) * T + t) * W + i] = up[t][i];
  depth[static_cast<int64_t>(blockIdx.x) * T + t] = n - 1;
}

// ---------------------------------------------------------------------------
// Kept rows.  A workgroup takes 64 bytes (or one scale) of every row of a (sequence,
// head, array): it reads the rows asked for, all of them, before it writes any, so the
// order and repetitions of the indexes do not matter.
// ---------------------------------------------------------------------------
template <typename X>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a, int slices) {
  constexpr int LPR = 4, RPP = 256 / LPR, PASSES = kMostTokens / RPP;  // X a lane, rows a pass
  const int slice = blockIdx.x % slices, bh = blockIdx.x / slices, which = blockIdx.y;
  const int b = bh / a.H, h = bh - b * a.H;
  const int col = (slice * LPR + threadIdx.x % LPR) * static_cast<int>(sizeof(X));
  if (a.data[which] == nullptr) return;
  const bool in = col < a.bytes[which];
  char *base = a.data[which] + b * a.s0[which] + h * a.s1[which] + a.first * a.s2[which] + col;
  X x[PASSES];
  int64_t from[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * RPP + threadIdx.x / LPR;
    from[i] = -1;
    if (in && r < a.n) {
      const int64_t at = static_cast<int64_t>(b) * a.n + r;
      from[i] = a.index_bytes == 8 ? static_cast<const int64_t *>(a.index)[at] : static_cast<const int32_t *>(a.index)[at];
      if (from[i] < 0 || from[i] >= a.limit) from[i] = -1;
    }
    if (from[i] >= 0) x[i] = *reinterpret_cast<const X *>(base + from[i] * a.s2[which]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * RPP + threadIdx.x / LPR;
    if (from[i] >= 0) *reinterpret_cast<X *>(base + r * a.s2[which]) = x[i];
  }
}

struct CachedPlan {
  int wr, groups, ns, gap, run, splits;
  bool nt;
};

CachedPlan plan_cached(const CachedProblem &p) {
  CachedPlan s;
  const int R = p.Hq / p.Hkv * p.T;
  // Waves alone read a tile once for each 32 rows, from L2 after the first, and meet no
  // barrier; waves that share read it once and pay where the matrix instructions fill the
  // chip: 24 tokens of 4 query heads over 8192 keys, 256 heads of 128 265 us alone and 193
  // shared, 63 tokens, 128 heads 257 and 182; 32 heads of 2048 keys, 16 tokens 18 and 25,
  // 63 tokens 28 and 30.  Codes and fp32 gain nothing from sharing (64 heads, 12 tokens
  // over 8192 codes 50 and 97 us; fp32, 16 over 4096 keys 103 and 182).
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv;
  const bool share = R > 32 && !p.q8 && p.dtype != TSATTN_F32 && heads * ((R + 127) / 128) >= 128;
  s.wr = share ? 4 : 1;
  s.groups = (R + 32 * s.wr - 1) / (32 * s.wr);
  const int tiles = (p.n + BN - 1) / BN;
  // the first key that some row's window holds (depth 0's)
  const int64_t low = p.window ? static_cast<int64_t>(p.n) - p.T - p.window + 1 : 0;
  const int first = low > 0 ? static_cast<int>(low) / BN : 0;
  const int sunk = p.window ? (p.sinks + BN - 1) / BN : 0;
  s.ns = sunk < first ? sunk : first;
  s.gap = first - s.ns;
  s.run = tiles - s.gap;
  // A wave for each SIMD: a second one costs a few tokens over 16 or 32 bits more in partial
  // results (step of 32 sequences, window 4096 of 8 heads of 128, through the memory-side
  // cache: 96 us, with two 102).
  // Codes, and rows enough for several waves, keep a SIMD busy beside the loads, and take
  // two where the parts stay few (63 tokens of 16 sequences over 8000 keys, 8 heads of 128:
  // 241 us in one part, 204 in two; 16 heads, 24 tokens of 7 sequences, codes: 38 us in 9
  // parts, 40 in 18).  A wave has 4 tiles or more to itself, of slower f32 ones 2 (17
  // tokens over 900 keys, 4 heads of 32: 18 us with 4, 14 with 2).
  const int64_t base = heads * s.groups;
  const int waves = s.wr > 1 ? s.wr : 64 * p.D * (p.dtype == TSATTN_F32 ? 4 : 2) <= 16384 ? 4 : 2;
  int64_t n = 1024 / waves / base;
  if (n < 1) n = 1;
  if (n <= 2 && (p.q8 || s.wr > 1)) n *= 2;
  const int least = (p.dtype == TSATTN_F32 ? 2 : 4) * (s.wr > 1 ? 1 : waves);
  if (n > s.run / least) n = s.run / least;
  s.splits = n < 1 ? 1 : static_cast<int>(n);
  // What is read once and is more than the memory-side cache's 256 MB passes it by: that
  // step, 537 MB, 96 -> 83 us; 268 MB 52 -> 51; of less, a cache that the step before has
  // left there is found again (34 MB: 15 us, read past it 17).
  const int64_t row = static_cast<int64_t>(p.D) * (p.q8 ? 1 : p.dtype == TSATTN_F32 ? 4 : 2);
  s.nt = s.groups == 1 && heads * s.run * BN * row * 2 > (int64_t(256) << 20);
  return s;
}

template <typename T, int D, bool Q8, bool NT>
void launch_kernel(const CachedArgs &a, int wr, dim3 grid, hipStream_t st) {
  if constexpr (!Q8 && !std::is_same_v<T, float>)
    if (wr == 4) return cached_kernel<T, D, Q8, 4, NT><<<grid, dim3(256), 0, st>>>(a);
  cached_kernel<T, D, Q8, 1, NT><<<grid, dim3(64 * kWaves<T, D, 1>), 0, st>>>(a);
}

template <typename T, int D, bool Q8>
void launch_wr(const CachedArgs &a, const CachedPlan &s, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hkv * a.splits * a.groups));
  if (s.nt) launch_kernel<T, D, Q8, true>(a, s.wr, grid, st);
  else launch_kernel<T, D, Q8, false>(a, s.wr, grid, st);
  if (a.splits > 1) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.R;
    constexpr int RPB = 256 / (D / 4);
    cached_merge_kernel<T, D><<<dim3(static_cast<unsigned>((rows + RPB - 1) / RPB)), dim3(256), 0, st>>>(a);
  }
}

template <typename T, bool Q8>
void launch_dim(const CachedArgs &a, int D, const CachedPlan &s, hipStream_t st) {
  if (D == 32) launch_wr<T, 32, Q8>(a, s, st);
  else if (D == 64) launch_wr<T, 64, Q8>(a, s, st);
  else if (D == 128) launch_wr<T, 128, Q8>(a, s, st);
  else if constexpr (!std::is_same_v<T, float>) launch_wr<T, 256, Q8>(a, s, st);
}

}  // namespace

bool cached_supported(const CachedProblem &p) {
  if (p.dtype == TSATTN_F32) return !p.q8 && (p.D == 32 || p.D == 64 || p.D == 128);
  return (p.dtype == TSATTN_F16 || p.dtype == TSATTN_BF16) && (p.D == 32 || p.D == 64 || p.D == 128 || p.D == 256);
}

size_t cached_workspace_bytes(const CachedProblem &p) {
  const CachedPlan s = plan_cached(p);
  return s.splits < 2 ? 0 : static_cast<size_t>(s.splits) * p.B * p.Hq * p.T * (p.D + 2) * sizeof(float);
}

hipError_t launch_cached(const CachedProblem &p, View q, View k, View v, View ks, View vs, View o, float *ws,
                         hipStream_t st) {
  const CachedPlan s = plan_cached(p);
  CachedArgs a{};
  a.B = p.B, a.Hkv = p.Hkv, a.rep = p.Hq / p.Hkv, a.T = p.T, a.n = p.n, a.R = a.rep * p.T;
  a.q = q, a.k = k, a.v = v, a.o = o, a.ks = ks, a.vs = vs;
  a.words = p.words, a.depth = p.depth, a.tree_rows = p.tree_rows, a.W = (p.T + 31) / 32;
  a.window = p.window, a.sinks = p.sinks;
  a.ns = s.ns, a.gap = s.gap, a.run = s.run, a.splits = s.splits, a.groups = s.groups;
  a.sl = static_cast<float>(p.scale) * kLog2e;
  a.rope = p.rope;
  a.ws = ws;
  Probe pr_(p.words ? "cached_tree" : "cached_window", st);
  if (p.dtype == TSATTN_F32) launch_dim<float, false>(a, p.D, s, st);
  else if (p.dtype == TSATTN_F16) p.q8 ? launch_dim<f16, true>(a, p.D, s, st) : launch_dim<f16, false>(a, p.D, s, st);
  else p.q8 ? launch_dim<bf16, true>(a, p.D, s, st) : launch_dim<bf16, false>(a, p.D, s, st);
  return hipGetLastError();
}

hipError_t launch_draft_tree(int trees, int T, const int32_t *parents, uint32_t *words, int32_t *depth, hipStream_t st) {
  Probe pr_("draft_tree", st);
  draft_tree_kernel<<<dim3(trees), dim3(kMostTokens), 0, st>>>(T, parents, words, depth);
  return hipGetLastError();
}

// Kept rows' pieces, as wide as every array's rows and addresses allow.
struct KeepPlan {
  int arrays, piece, slices;
};
static KeepPlan plan_keep(const KeepArgs &a) {
  int arrays = 0, most = 0;
  uintptr_t all = 0;
  for (int i = 0; i < 4; ++i)
    if (a.data[i]) {
      arrays = i + 1;
      most = a.bytes[i] > most ? a.bytes[i] : most;
      if (i < 2)
        all |= reinterpret_cast<uintptr_t>(a.data[i]) | static_cast<uintptr_t>(a.bytes[i]) |
               static_cast<uintptr_t>(a.s0[i]) | static_cast<uintptr_t>(a.s1[i]) | static_cast<uintptr_t>(a.s2[i]);
    }
  if (arrays > 2 && all % 16 == 0) all |= 4;  // (scales: 4 bytes a row)
  const int piece = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
  return KeepPlan{arrays, piece, most / (4 * piece) + (most % (4 * piece) != 0)};
}

int64_t keep_groups(const KeepArgs &a) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.H;
  return heads < (int64_t(1) << 31) ? heads * plan_keep(a).slices : heads;
}

hipError_t launch_keep(const KeepArgs &a, hipStream_t st) {
  const KeepPlan s = plan_keep(a);
  Probe pr_("cache_keep", st);
  const dim3 grid(static_cast<unsigned>(keep_groups(a)), s.arrays);
  if (s.piece == 16) keep_kernel<u32x4><<<grid, dim3(256), 0, st>>>(a, s.slices);
  else if (s.piece == 4) keep_kernel<uint32_t><<<grid, dim3(256), 0, st>>>(a, s.slices);
  else keep_kernel<uint8_t><<<grid, dim3(256), 0, st>>>(a, s.slices);
  return hipGetLastError();
}

}  // namespace tsattn
