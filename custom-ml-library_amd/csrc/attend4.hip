// Attention over the 4-bit paged cache (pages4.h): a few query rows per KV head
// against every cached position, split over the positions and merged.
//
// Math.  With q's parts and the codes' levels c exact in bf16 and fp32 sums,
//   S[j] = sum_s sk[j, s] (q_s . c_j,s),   P = softmax of scale S,
//   O_s = sum_j (P[j] sv[j, s]) c_j,s      for each group s of 32 channels:
// the scales stay outside the matrix products, so no dequantised value is formed.
// Where a KV head has few rows, the groups take columns of the 16-wide B operand beside
// them: column c = G r + s holds row r's group s, zero in the other groups' channels.
// One chain of MFMAs then sums each group of each row by itself, a score takes one
// multiply by its key's scale and a sum over G neighbouring lanes, and the value product
// takes P sv of its own column: a lane scales 8 probabilities a tile where it would
// scale 8 G otherwise.  The price is in MFMAs, which have time (a value block is
// multiplied for all columns and used by those of its group).  Where there are many
// (WIDE), a column is a row, and the scales multiply the groups' scores, and the
// probabilities, one group after the other; they reach the lanes from the one that
// loaded them.
//
// Precision.  q enters exactly: bf16 in one part, f16 in two, fp32 in three.  P sv
// enters as two bf16 parts (within 2^-16 of each: the first is truncated), for fp32 as
// three (exactly).
//
// A wave works alone on every fourth or eighth tile of its split, two tiles ahead in
// registers, straight from memory in operand order (pages4.h); waves merge in LDS,
// splits in a second kernel where there is more than one.
//
// Bounds.  Large calls by memory: 64 sequences of 32 heads over up to 8192 positions
// (bf16, D128), 1.30 GB, 203 us with the merge: 6.4 TB/s, at 22% of the matrix cores'
// time and 56% of the vector units'.  Middling ones by the start of a workgroup and a
// tile's latency: 64 x 8 KV heads over 1025, 4 rows (f16, D128), 77 MB, 18.4 us, of
// which 4 pass before the second tile.  Small ones by latency alone: 8 heads over 200,
// 4 us.  Many rows by the vector units (levels, scales, roundings: about 320 instructions
// a tile of 32 positions and 16 rows of bf16 D128).
#include "pages4.h"
#include "rope_math.h"

namespace tsattn {
namespace {

// Positions a split at most: 32 tiles a wave of four, whose lanes hold their page numbers.
constexpr int kMostSplit = 4096;
static_assert(kMostSplit / kTile / 4 <= 64, "one lane a tile");

template <typename T>
constexpr int q_parts() { return std::is_same_v<T, bf16> ? 1 : std::is_same_v<T, f16> ? 2 : 3; }
template <typename T>
constexpr int p_parts() { return std::is_same_v<T, float> ? 3 : 2; }

// Two floats as N pairs of bf16 whose sums they are: all but the last truncated.
// (A subtraction contracted with the product before it would keep a scale from being
// that product's own operand.)
template <int N>
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t (&out)[N]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    out[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    a -= __builtin_bit_cast(float, x & 0xFFFF0000u);
    b -= __builtin_bit_cast(float, y & 0xFFFF0000u);
  }
  out[N - 1] = pack2<bf16>(a, b);
}

// Sum of a x over the G neighbouring lanes of a row's groups.  (Contracted, the first
// addition would take a multiply-add and a move of its own from the other lane.)
template <int G>
__device__ __forceinline__ float scaled_sum(float a, float x) {
#pragma clang fp contract(off)
  auto dpp = [](float v, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  float y = a * x;
  if constexpr (G >= 2) y += dpp(y, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  if constexpr (G >= 4) y += dpp(y, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  if constexpr (G >= 8) y += dpp(y, std::integral_constant<int, 0x141>{});  // half-row mirror: the other quad
  return y;
}

// The value of lane S of the 16 that share a lane's g.
template <int S>
__device__ __forceinline__ float from_lane(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x150 + S, 0xF, 0xF, true));  // row_newbcast
}

// f(integral constants 0 .. N - 1).
template <int N, typename F>
__device__ __forceinline__ void each(F &&f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// A lane's share of a tile: codes of keys and values, eight scales of each.
template <int G>
struct Held {
  using Chunk = std::conditional_t<G == 1, u32x2, u32x4>;
  static constexpr int N = G == 1 ? 1 : G / 2;
  Chunk k[N], v[N];
  u32x4 ks, vs;
  __device__ __forceinline__ uint32_t kw(int w) const { return G == 1 ? k[0][w] : k[w >> 2][w & 3]; }
  __device__ __forceinline__ uint32_t vw(int w) const { return G == 1 ? v[0][w] : v[w >> 2][w & 3]; }
};

template <typename T, int G, int NB, int NWV, bool WIDE>
__global__ __launch_bounds__(64 * NWV, (G == 8 && (WIDE || std::is_same_v<T, float>) ? 1 : 2)) void attend4_kernel(Attend4 a) {
  constexpr int D = 32 * G, W = 2 * G, NQ = q_parts<T>(), NP = p_parts<T>();
  constexpr int RB = WIDE ? 16 : 16 / G, ROWS = RB * NB;  // rows a column block, a workgroup
  constexpr int PIECES = WIDE ? G : 1;                    // of a row that a lane holds
  constexpr int MR = WIDE ? 16 : ROWS, MD = WIDE && D > 128 ? 128 : D;  // rows, channels merged at a time
  constexpr int LD = MD + 4;                              // (rows of the merge start in different banks)
  __shared__ __attribute__((aligned(16))) float part[NWV][MR][LD];
  __shared__ float state[NWV][ROWS][2];  // their maximum and sum

  const int b = blockIdx.z, split = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rl = WIDE ? c : c / G, grp = c % G;  // the lane's row in its column block, its group
  const int len = a.s.len[b], trow = a.s.row[b];
  const int hk = a.blocks == 1 ? blockIdx.x : blockIdx.x / a.blocks;
  const int row0 = a.first + (blockIdx.x - hk * a.blocks) * ROWS;
  const int begin = split * a.split;
  const int live_rows = min(ROWS, a.first + a.rows - row0);
  auto out_row = [&](int r) __attribute__((always_inline)) {
    const int rr = fdiv(row0 + r, a.by_len_q), qi = row0 + r - rr * a.len_q;
    return static_cast<T *>(const_cast<void *>(a.o.data)) + b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
           qi * a.o.s2;
  };
  if (begin >= len) {  // no positions here: an empty sequence's rows are zero
    if (a.splits == 1)
      for (int r = w; r < live_rows; r += NWV)
        for (int d = lane; d < D; d += 64) out_row(r)[d] = static_cast<T>(0.f);
    return;
  }
  const int keys = min(a.split, len - begin);
  const int n_tiles = (keys + kTile - 1) / kTile;
  const int mine = n_tiles > w ? (n_tiles - 1 - w) / NWV + 1 : 0;
  const int tile0 = begin / kTile + w;

  // the queries' rows, on their way first: row r of the block, channels 32 grp + 8 g .. + 7
  constexpr int QW = sizeof(T) / 2;  // 16-byte loads a row piece
  u32x4 raw[NB][PIECES][QW];
  int qpos[NB];  // the row's query's number
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = nb * RB + rl < live_rows ? row0 + nb * RB + rl : row0;
    const int rr = fdiv(r, a.by_len_q);
    qpos[nb] = r - rr * a.len_q;
    const T *qp = static_cast<const T *>(a.q.data) + b * a.q.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.q.s1 +
                  qpos[nb] * a.q.s2 + (WIDE ? 0 : 32 * grp) + 8 * g;
#pragma unroll
    for (int e = 0; e < PIECES; ++e)
#pragma unroll
      for (int i = 0; i < QW; ++i) raw[nb][e][i] = reinterpret_cast<const u32x4 *>(qp + 32 * e)[i];
  }
  // the wave's page numbers, lane t's for its tile t: one load, and none in the loop
  // (lanes past the wave's tiles: the split's last, as the table need not go on)
  const int ids = a.p.table[trow * a.p.stride + ((begin / kTile + min(w + NWV * lane, n_tiles - 1)) >> a.p.per_page)];
  auto load = [&](Held<G> &x, int t) __attribute__((always_inline)) {
    using C = typename Held<G>::Chunk;
    const char *base = tile4_at(a.p, static_cast<uint32_t>(__builtin_amdgcn_readlane(ids, t)), tile0 + NWV * t, hk);
#pragma unroll
    for (int q = 0; q < Held<G>::N; ++q) {
      x.k[q] = __builtin_nontemporal_load(reinterpret_cast<const C *>(base) + 64 * q + lane);
      x.v[q] = __builtin_nontemporal_load(reinterpret_cast<const C *>(base + 16 * D) + 64 * q + lane);
    }
    x.ks = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + 32 * D) + g * G + grp);
    x.vs = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + 34 * D) + g * G + grp);
  };
  Held<G> x0, x1;
  if (mine > 0) load(x0, 0);
  if (mine > 1) load(x1, 1);

  // the B operand: the row's pieces in their k-steps; of a lane's one piece, zero in the others
  u32x4 qf[NB][NQ][G];
  int klim[NB];  // positions of the split that the row sees: [0, klim)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const bool live = nb * RB + rl < live_rows;
    const int at = len - a.len_q + qpos[nb];  // the query's position
    klim[nb] = a.causal ? min(keys, at + 1 - begin) : keys;
#pragma unroll
    for (int piece = 0; piece < PIECES; ++piece) {
      T x[8];
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        const T *e = reinterpret_cast<const T *>(&raw[nb][piece][i]);
#pragma unroll
        for (int j = 0; j < 8 / QW; ++j) x[i * (8 / QW) + j] = e[j];
      }
      if (a.cos) {
        const int64_t e = static_cast<int64_t>(max(at, 0)) * (D / 2) + 16 * (WIDE ? piece : grp) + 4 * g;
        T cw[4], sw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) cw[i] = static_cast<const T *>(a.cos)[e + i], sw[i] = static_cast<const T *>(a.sin)[e + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate_pair(x[2 * i], x[2 * i + 1], cw[i], sw[i], false);
      }
      uint32_t pt[NQ][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t two[NQ];
        split_bf16<NQ>(live ? static_cast<float>(x[2 * i]) * a.sign : 0.f,
                       live ? static_cast<float>(x[2 * i + 1]) * a.sign : 0.f, two);
#pragma unroll
        for (int n = 0; n < NQ; ++n) pt[n][i] = two[n];
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 y{pt[n][0], pt[n][1], pt[n][2], pt[n][3]};
        if constexpr (WIDE) {
          qf[nb][n][piece] = y;
        } else {
#pragma unroll
          for (int ks = 0; ks < G; ++ks) qf[nb][n][ks] = ks == grp ? y : u32x4{0, 0, 0, 0};
        }
      }
    }
  }
  // tiles before `edge` are seen whole by every row
  const int edge = (a.causal ? min(keys, len - a.len_q + 1 - begin) : keys) / kTile;

  f32x4 oacc[NB][W];
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY, l[nb] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) oacc[nb][i] = f32x4{};
  }

  // Chains of dependent MFMAs alternate: the two halves of the scores (WIDE: of each
  // group), pairs of value blocks.
  auto compute = [&](const Held<G> &t4, int t) __attribute__((always_inline)) {
    const int tile = w + NWV * t;  // of the split
    float ksc[8], vsc[8];  // the scales of the lane's group, keys 4 g .. + 3 and 16 + 4 g .. + 3
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      ksc[i] = __builtin_bit_cast(float, t4.ks[i >> 1] << 16);
      ksc[i + 1] = __builtin_bit_cast(float, t4.ks[i >> 1] & 0xFFFF0000u);
      vsc[i] = __builtin_bit_cast(float, t4.vs[i >> 1] << 16);
      vsc[i + 1] = __builtin_bit_cast(float, t4.vs[i >> 1] & 0xFFFF0000u);
    }
    float x[NB][8];  // the scores
    if constexpr (WIDE) {
      each<G>([&](auto group) __attribute__((always_inline)) {
        constexpr int ks = decltype(group)::value;
        f32x4 s[NB][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const u32x4 kf = levels_bf16(t4.kw(kb * G + ks));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            s[nb][kb] = f32x4{};
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[nb][kb] = mfma16<bf16>(kf, qf[nb][n][ks], s[nb][kb]);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float sc = from_lane<ks>(ksc[i]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            x[nb][i] = ks == 0 ? s[nb][i >> 2][i & 3] * sc : fmaf(s[nb][i >> 2][i & 3], sc, x[nb][i]);
        }
      });
    } else {
      f32x4 s[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = f32x4{};
#pragma unroll
      for (int ks = 0; ks < G; ++ks) {
        u32x4 kf[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) kf[kb] = levels_bf16(t4.kw(kb * G + ks));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[nb][kb] = mfma16<bf16>(kf[kb], qf[nb][n][ks], s[nb][kb]);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[nb][i] = scaled_sum<G>(s[nb][i >> 2][i & 3], ksc[i]);
    }
    const bool whole = tile < edge;
    u32x4 pb[NB][NP];
    float pr[NB][8];   // WIDE: the probabilities
    uint32_t seen[NB]; // and, of a tile that is not whole, which the row sees
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i] = vsc[i];
      seen[nb] = 0xFFu;
      if (!whole) {  // what a row does not see weighs nothing, whatever its scales are
        const int lim = klim[nb] - tile * kTile - 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (16 * (i >> 2) + (i & 3) >= lim) x[nb][i] = -INFINITY, vs[i] = 0.f, seen[nb] &= ~(1u << i);
      }
      float mx = x[nb][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[nb][i]);
      mx = quad_row_max(mx) * a.sl;  // (sl > 0)
      if (__ballot(mx > m[nb]) != 0ull) {
        const float mn = fmaxf(m[nb], mx);
        const float corr = mn == -INFINITY ? 1.f : fast_exp2(m[nb] - mn);
        m[nb] = mn;
        l[nb] *= corr;
#pragma unroll
        for (int i = 0; i < W; ++i) oacc[nb][i] *= corr;
      }
      const float base = m[nb] == -INFINITY ? 0.f : -m[nb];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float p0 = fast_exp2(fmaf(x[nb][i], a.sl, base)), p1 = fast_exp2(fmaf(x[nb][i + 1], a.sl, base));
        l[nb] += p0 + p1;
        pr[nb][i] = p0, pr[nb][i + 1] = p1;
        uint32_t two[NP];
        split_bf16<NP>(p0 * vs[i], p1 * vs[i + 1], two);
#pragma unroll
        for (int n = 0; n < NP; ++n) pb[nb][n][i >> 1] = two[n];
      }
    }
    if constexpr (WIDE) {  // the probabilities times one group's scales after the other's
      auto values = [&](auto every) __attribute__((always_inline)) {
        each<G>([&](auto group) __attribute__((always_inline)) {
          constexpr int s = decltype(group)::value;
          const u32x4 vf[2] = {levels_bf16(t4.vw(2 * s)), levels_bf16(t4.vw(2 * s + 1))};
          float y[8];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y[i] = pr[nb][i] * from_lane<s>(vsc[i]);
              if (!decltype(every)::value) y[i] = seen[nb] >> i & 1 ? y[i] : 0.f;
            }
            u32x4 ps[NP];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              uint32_t two[NP];
              split_bf16<NP>(y[i], y[i + 1], two);
#pragma unroll
              for (int n = 0; n < NP; ++n) ps[n][i >> 1] = two[n];
            }
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) oacc[nb][2 * s + e] = mfma16<bf16>(vf[e], ps[n], oacc[nb][2 * s + e]);
          }
        });
      };
      if (whole) values(std::true_type{});
      else values(std::false_type{});
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const u32x4 vf[2] = {levels_bf16(t4.vw(i)), levels_bf16(t4.vw(i + 1))};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int n = 0; n < NP; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) oacc[nb][i + e] = mfma16<bf16>(vf[e], pb[nb][n], oacc[nb][i + e]);
      }
    }
  };

  for (int t = 0; t < mine; t += 2) {
    compute(x0, t);
    if (t + 2 < mine) load(x0, t + 2);
    if (t + 1 < mine) {
      compute(x1, t + 1);
      if (t + 3 < mine) load(x1, t + 3);
    }
  }

  // Merge the waves, MR rows and MD channels at a time.  Lane (c, g) has row rl's
  // channels 16 i + 4 g .. + 3 (for the blocks i of its group, unless WIDE); then a wave
  // sums a row over the waves, PER channels a lane.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float lt = l[nb] + __shfl_xor(l[nb], 16, 64);
    lt += __shfl_xor(lt, 32, 64);
    if (g == 0 && (WIDE || grp == 0)) {
      state[w][nb * RB + rl][0] = m[nb];
      state[w][nb * RB + rl][1] = lt;
    }
  }
  constexpr int PER = MD < 64 ? 1 : MD / 64;
  using Piece = std::conditional_t<PER == 1, float, std::conditional_t<PER == 2, f32x2, f32x4>>;
#pragma unroll
  for (int r0 = 0; r0 < ROWS; r0 += MR) {
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += MD) {
      if (r0 + d0 > 0) __syncthreads();  // (the rows and channels before are read)
#pragma unroll
      for (int nb = r0 / RB; nb < (r0 + MR) / RB; ++nb) {
        float *to = part[w][nb * RB - r0 + rl];
#pragma unroll
        for (int i = 0; i < MD / 16; ++i)
          if (WIDE || i / 2 == grp) *reinterpret_cast<f32x4 *>(to + 16 * i + 4 * g) = oacc[nb][d0 / 16 + i];
      }
      __syncthreads();
      for (int r = r0 + w; r < min(r0 + MR, live_rows); r += NWV) {
        float mv[NWV], M = -INFINITY, total = 0.f, sum[PER] = {};
        Piece x[NWV];
#pragma unroll
        for (int v = 0; v < NWV; ++v) {
          mv[v] = state[v][r][0];
          x[v] = *reinterpret_cast<const Piece *>(part[v][r - r0] + (MD < 64 ? lane & (MD - 1) : PER * lane));
        }
#pragma unroll
        for (int v = 0; v < NWV; ++v) M = fmaxf(M, mv[v]);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int v = 0; v < NWV; ++v) {
          const float f = fast_exp2(mv[v] - base);
          const float *e = reinterpret_cast<const float *>(&x[v]);
          total = fmaf(state[v][r][1], f, total);
#pragma unroll
          for (int i = 0; i < PER; ++i) sum[i] = fmaf(e[i], f, sum[i]);
        }
        if (lane * PER < MD) {
          const int d = d0 + PER * lane;
          if (a.splits > 1) {
            float *to = a.ws + ((static_cast<int64_t>(b * a.p.heads + hk) * a.splits + split) * a.rows + row0 - a.first + r) *
                                   (D + 2);
#pragma unroll
            for (int i = 0; i < PER; ++i) to[d + i] = sum[i];
            if (d == 0) to[D] = M, to[D + 1] = total;
          } else {
            T *to = out_row(r);
#pragma unroll
            for (int i = 0; i < PER; ++i) to[d + i] = static_cast<T>(total == 0.f ? 0.f : sum[i] / total);
          }
        }
      }
    }
  }
}

// One wave an output row: the splits' partial states rescaled to their largest
// maximum, 16 splits' loads in flight.
template <typename T, int D>
__global__ __launch_bounds__(64) void attend4_merge_kernel(Attend4 a) {
  const int lane = threadIdx.x, b = blockIdx.z, hk = blockIdx.y, r = blockIdx.x;
  const int n = (a.s.len[b] + a.split - 1) / a.split;
  const float *base = a.ws + (static_cast<int64_t>(b * a.p.heads + hk) * a.splits * a.rows + r) * (D + 2);
  const int64_t stride = static_cast<int64_t>(a.rows) * (D + 2);
  constexpr int PER = (D + 63) / 64, U = 16;
  float acc[PER] = {}, L = 0.f, M = -INFINITY;
  for (int s0 = 0; s0 < n; s0 += U) {
    float ms[U], ls[U], x[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float *from = base + min(s0 + u, n - 1) * stride;
      ms[u] = from[D], ls[u] = from[D + 1];
#pragma unroll
      for (int i = 0; i < PER; ++i) x[u][i] = from[min(lane + 64 * i, D - 1)];
    }
    const float before = M;
#pragma unroll
    for (int u = 0; u < U; ++u) M = fmaxf(M, ms[u]);
    const float at = M == -INFINITY ? 0.f : M, corr = fast_exp2(before - at);
    L *= corr;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] *= corr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float e = s0 + u < n ? fast_exp2(ms[u] - at) : 0.f;  // (the last split again: finite, or NaN as it is)
      L = fmaf(ls[u], e, L);
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = fmaf(x[u][i], e, acc[i]);
    }
  }
  const int rr = fdiv(a.first + r, a.by_len_q), qi = a.first + r - rr * a.len_q;
  T *out = static_cast<T *>(const_cast<void *>(a.o.data)) + b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
           qi * a.o.s2;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < D) out[lane + 64 * i] = static_cast<T>(L == 0.f ? 0.f : acc[i] / L);
}

}  // namespace

// How a workgroup is made -- columns of groups, one block of them or two, with four
// waves (two or three workgroups a CU) or eight, which take a CU by themselves; or
// columns of rows with four -- and splits: those that a model of the time likes best.
// Two blocks read the cache once for twice the rows; one, where the memory is not what
// a call waits for, has twice the workgroups.  In us: a workgroup's prologue and merge
// 2.4 or 2.6, of rows 3.9 to 6.3; a tile of a wave the largest of its own latency (by
// its products; bf16 D128 1.0 with one block, 2.1 with two, 1.1 of rows; fp32 D128 1.8,
// of rows 1.3; bf16 D256 1.9, of rows 2.0), of the issue slots of the waves beside it and
// of the memory's rate; where the workgroups do not fit the chip at once, their rounds
// over it; the second kernel 3.4.  Its constants are fitted to 104 shapes, of which it
// takes 3% longer than the best choice in the mean (groups alone 34%, for the 70 with
// more rows than one block).  Measured, what it picks and another: 7 sequences of 4 KV
// heads up to 4001, 20 rows of bf16 D128: rows 14.4, groups in one block 17.4, in two
// 19.1; 8 of 8 heads over 8000, 16 rows: rows 27, groups 44; 4 of 32 heads over 4000, f16
// D128: eight waves and 2 splits 19.0, four and 3 22.4; 3 of one head over 1500, fp32
// D128: 12 splits 7.1, one 13.1; 64 of 8 heads over 1025, 4 rows of f16 D128: one split
// 18.5, three 24.
void plan_attend4(Attend4 *a, int dtype, const int32_t *lens) {
  int64_t total = 0;
  int longest = 1;
  for (int i = 0; i < a->n; ++i) {
    total += lens[i];
    longest = lens[i] > longest ? lens[i] : longest;
  }
  const int dim = a->p.dim;
  const int parts = dtype == TSATTN_F32 ? 6 : dtype == TSATTN_F16 ? 4 : 3;
  const int fewest = (longest + kMostSplit - 1) / kMostSplit;
  double best = 1e30;
  for (int waves = 4; waves <= 8; waves += 4) {
    if (waves == 8 && dtype != TSATTN_BF16 && dim == 256) continue;  // (more registers than eight waves have)
    const int unit = kTile * waves;
    for (int k : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      const int n = k > fewest ? k : fewest;
      int even = ((longest + n - 1) / n + unit - 1) / unit * unit;
      if (n > 1 && even < kMostSplit) even = (even / 128 | 1) * 128;
      if (k > 1 && (k <= fewest || even < 128 || n > longest)) continue;
      int live = 0;
      if (total == static_cast<int64_t>(a->n) * longest) {
        live = a->n * ((longest + even - 1) / even);
      } else {
        const float per_split = 1.f / even;
        for (int i = 0; i < a->n; ++i) live += 1 + static_cast<int>(static_cast<float>(lens[i] - 1) * per_split);
      }
      const double tiles = static_cast<double>(even < longest ? even : longest) / unit;
      for (int make = 0; make < 3; ++make) {
        const bool wide = make == 2;
        const int nb = make == 1 ? 2 : 1, one_block = 512 / dim;
        if (make && a->rows <= one_block) break;
        // (two blocks' operands are more registers than fp32 queries, three parts, and 256 channels leave)
        if (make == 1 && (dtype == TSATTN_F32 || dim == 256)) continue;
        if (wide && (waves == 8 || dim == 32)) continue;  // (32 channels: a row is one group)
        const int per = wide ? 16 : one_block * nb, blocks = (a->rows + per - 1) / per;
        const double latency = wide ? 0.33 + dim / 32 * (0.17 + 0.011 * parts)
                                    : nb * (0.21 + dim / 16 * (0.008 + 0.032 * parts));
        const double start = wide ? 3.1 + 0.4 * (dim / 32) : waves == 8 ? 2.6 : 2.4;
        const double slots = waves == 8 || (wide && dim == 256)             ? 256.
                             : nb == 2 || dim == 256 || (wide && dim == 128) ? 512.
                                                                            : 768.;
        const double groups = static_cast<double>(a->p.heads) * blocks, wgs = groups * live, rounds = wgs / slots;
        const double busy = (wgs < slots ? wgs : slots) * waves;
        const double rate = busy * 36 * dim / 7.4e6, issue = (wide ? 0.69 : 0.55) * latency * busy / 1024;
        const double alone = latency > issue ? latency : issue;
        const double one = start + (tiles > 1 ? tiles : 1) * (alone > rate ? alone : rate);
        double cost = one;
        if (rounds > 3) {
          const double sum = groups * total / unit, most = wgs * start + sum * alone;
          cost = ((most > sum * rate ? most : sum * rate) + (wide ? 0.83 : 0.05) * wgs * start) / slots +
                 (wide ? 0.02 : 0.14) * one;
        } else if (rounds > 1) {
          cost = one * (wide ? 1.1 * rounds : 1.3 + 0.62 * (rounds - 1));
        }
        if (n > 1) cost += 2.9 + 0.5 * ((n + 15) / 16) + 8. * a->n * a->p.heads * n * a->rows * (dim + 2) / 7.4e6;
        if (cost < best) {
          best = cost;
          a->wide = wide, a->columns = nb, a->blocks = blocks, a->waves = waves;
          a->split = even, a->splits = (longest + even - 1) / even;
        }
      }
    }
  }
}

hipError_t launch_attend4(const Attend4 &a, int dtype, hipStream_t st) {
  const int dim = a.p.dim;
  const dim3 grid(a.p.heads * a.blocks, a.splits, a.n);
  auto launch = [&](auto t, auto g) {
    using T = decltype(t);
    constexpr int G = decltype(g)::value;
    constexpr bool f32 = std::is_same_v<T, float>;
    {
      Probe pr_("attend4", st);
      auto run = [&](auto n) {
        constexpr int NB = decltype(n)::value;
        if constexpr (G < 8 || std::is_same_v<T, bf16>) {
          if (a.waves == 8) {
            attend4_kernel<T, G, NB, 8, false><<<grid, dim3(512), 0, st>>>(a);
            return;
          }
        }
        attend4_kernel<T, G, NB, 4, false><<<grid, dim3(256), 0, st>>>(a);
      };
      if (a.wide) {
        if constexpr (G > 1) attend4_kernel<T, G, 1, 4, true><<<grid, dim3(256), 0, st>>>(a);
      } else if constexpr (!f32 && G < 8) {
        if (a.columns == 2) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 1>{});
      } else {
        run(std::integral_constant<int, 1>{});
      }
    }
    if (a.splits > 1) {
      Probe pr_("attend4_merge", st);
      attend4_merge_kernel<T, 32 * G><<<dim3(a.rows, a.p.heads, a.n), dim3(64), 0, st>>>(a);
    }
  };
  auto dims = [&](auto t) {
    if (dim == 32) launch(t, std::integral_constant<int, 1>{});
    else if (dim == 64) launch(t, std::integral_constant<int, 2>{});
    else if (dim == 128) launch(t, std::integral_constant<int, 4>{});
    else launch(t, std::integral_constant<int, 8>{});
  };
  if (dtype == TSATTN_F32) dims(float{});
  else if (dtype == TSATTN_F16) dims(f16{});
  else dims(bf16{});
  return hipGetLastError();
}

}  // namespace tsattn
