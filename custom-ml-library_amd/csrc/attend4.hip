// Attention over the 4-bit paged cache (pages4.h): a few query rows per KV head
// against every cached position, split over the positions and merged.
//
// Math.  With q's parts and the codes' levels c exact in bf16 and fp32 sums,
//   S[j] = sum_s sk[j, s] (q_s . c_j,s),   P = softmax of scale S,
//   O_s = sum_j (P[j] sv[j, s]) c_j,s      for each group s of 32 channels:
// the scales stay outside the matrix products, so no dequantised value is formed.
// The groups take columns of the 16-wide B operand beside the rows: column
// c = G r + s holds row r's group s, zero in the other groups' channels.  One
// chain of MFMAs then sums each group of each row by itself, a score takes one
// multiply by its key's scale and a sum over G neighbouring lanes, and the value
// product takes P sv of its own column: a lane scales 8 probabilities a tile
// where it would scale 8 G otherwise.  The price is in MFMAs, which have time (a
// value block is multiplied for all columns and used by those of its group).
//
// Precision.  q enters exactly: bf16 in one part, f16 in two, fp32 in three. P sv
// enters as two bf16 parts (2^-17 of each), for fp32 as three (2^-25).
//
// A wave works alone on the tiles w, w + 4, ... of its split, two tiles ahead in
// registers, straight from memory in operand order (pages4.h); waves merge in LDS,
// splits in a second kernel where there is more than one.
#include "pages4.h"
#include "rope_math.h"

namespace tsattn {
namespace {

constexpr int NWV = 4;

template <typename T>
constexpr int q_parts() { return std::is_same_v<T, bf16> ? 1 : std::is_same_v<T, f16> ? 2 : 3; }
template <typename T>
constexpr int p_parts() { return std::is_same_v<T, float> ? 3 : 2; }

// Two floats as N pairs of bf16 whose sums they are: all but the last truncated.
template <int N>
__device__ __forceinline__ void split_bf16(float a, float b, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    out[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    a -= __builtin_bit_cast(float, x & 0xFFFF0000u);
    b -= __builtin_bit_cast(float, y & 0xFFFF0000u);
  }
  out[N - 1] = pack2<bf16>(a, b);
}

// Sum over the G neighbouring lanes of a row's groups.
template <int G>
__device__ __forceinline__ float group_sum4(float x) {
  auto dpp = [](float v, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  if constexpr (G >= 2) x += dpp(x, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  if constexpr (G >= 4) x += dpp(x, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  if constexpr (G >= 8) x += dpp(x, std::integral_constant<int, 0x141>{});  // half-row mirror: the other quad
  return x;
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

template <typename T, int G, int NB>
__global__ __launch_bounds__(64 * NWV, (std::is_same_v<T, float> && G == 8 ? 1 : 2)) void attend4_kernel(Attend4 a) {
  constexpr int D = 32 * G, W = 2 * G, NQ = q_parts<T>(), NP = p_parts<T>();
  constexpr int RB = 16 / G, ROWS = RB * NB;  // rows a column block, a workgroup
  __shared__ float part[NWV][ROWS][D + 2];

  const int b = blockIdx.z, split = blockIdx.y;
  const int blocks = (a.rows + ROWS - 1) / ROWS;
  const int hk = blockIdx.x / blocks, row0 = (blockIdx.x - hk * blocks) * ROWS;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rl = c / G, grp = c % G;  // the lane's row in its column block, its group
  const int len = a.s.len[b];
  const int begin = split * a.split;
  const int live_rows = min(ROWS, a.rows - row0);
  if (begin >= len) {  // no positions here: an empty sequence's rows are zero
    if (a.splits == 1)
      for (int i = tid; i < live_rows * D; i += 64 * NWV) {
        const int r = row0 + i / D, d = i % D, rr = r / a.len_q, qi = r - rr * a.len_q;
        static_cast<T *>(const_cast<void *>(a.o.data))[b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
                                                       qi * a.o.s2 + d] = static_cast<T>(0.f);
      }
    return;
  }
  const int keys = min(a.split, len - begin);
  const int n_tiles = (keys + kTile - 1) / kTile;
  const int mine = n_tiles > w ? (n_tiles - 1 - w) / NWV + 1 : 0;
  const int tile0 = begin / kTile + w;
  const int32_t *ids = a.p.table + a.s.row[b] * a.p.stride;

  // queries: row r of the block, channels 32 grp + 8 g .. + 7, in k-step grp
  u32x4 qf[NB][NQ][G];
  int klim[NB];  // positions of the split that the row sees: [0, klim)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = row0 + nb * RB + rl;
    const bool live = nb * RB + rl < live_rows;
    const int rr = live ? r / a.len_q : 0, qi = live ? r - rr * a.len_q : 0;
    const T *qp = static_cast<const T *>(a.q.data) + b * a.q.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.q.s1 +
                  qi * a.q.s2 + 32 * grp + 8 * g;
    T x[8];
    if constexpr (sizeof(T) == 2) {
      const u32x4 raw = ld16(qp);
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = e[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = qp[i];
    }
    const int at = max(len - a.len_q + qi, 0);  // the query's position
    if (a.cos) {
      const int64_t e = static_cast<int64_t>(at) * (D / 2) + 16 * grp + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rotate_pair(x[2 * i], x[2 * i + 1], static_cast<const T *>(a.cos)[e + i], static_cast<const T *>(a.sin)[e + i],
                    false);
    }
    klim[nb] = a.causal ? min(keys, len - a.len_q + qi + 1 - begin) : keys;
    uint32_t pt[NQ][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t two[NQ];
      split_bf16<NQ>(live ? static_cast<float>(x[2 * i]) : 0.f, live ? static_cast<float>(x[2 * i + 1]) : 0.f, two);
#pragma unroll
      for (int n = 0; n < NQ; ++n) pt[n][i] = two[n];
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int ks = 0; ks < G; ++ks)
        qf[nb][n][ks] = ks == grp ? u32x4{pt[n][0], pt[n][1], pt[n][2], pt[n][3]} : u32x4{0, 0, 0, 0};
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

  auto id_of = [&](int t) __attribute__((always_inline)) {
    return static_cast<uint32_t>(ids[(tile0 + NWV * min(t, mine - 1)) >> a.p.per_page]);
  };
  auto load = [&](Held<G> &x, int t, uint32_t id) __attribute__((always_inline)) {
    using C = typename Held<G>::Chunk;
    const char *base = tile4_at(a.p, id, tile0 + NWV * t, hk);
#pragma unroll
    for (int q = 0; q < Held<G>::N; ++q) {
      x.k[q] = __builtin_nontemporal_load(reinterpret_cast<const C *>(base) + 64 * q + lane);
      x.v[q] = __builtin_nontemporal_load(reinterpret_cast<const C *>(base + 16 * D) + 64 * q + lane);
    }
    x.ks = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + 32 * D) + g * G + grp);
    x.vs = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + 34 * D) + g * G + grp);
  };
  auto compute = [&](const Held<G> &t4, int t) __attribute__((always_inline)) {
    const int tile = w + NWV * t;  // of the split
    f32x4 s[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = f32x4{};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int ks = 0; ks < G; ++ks) {
        const u32x4 kf = levels_bf16(t4.kw(kb * G + ks));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[nb][kb] = mfma16<bf16>(kf, qf[nb][n][ks], s[nb][kb]);
      }
    u32x4 pb[NB][NP];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = group_sum4<G>(s[nb][i >> 2][i & 3] * from_bf16((t4.ks[i >> 1] >> (16 * (i & 1))) & 0xFFFFu)) * a.sl;
      if (tile >= edge) {
        const int lim = klim[nb] - tile * kTile - 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (16 * (i >> 2) + (i & 3) >= lim) x[i] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
      mx = quad_row_max(mx);
      if (__ballot(mx > m[nb]) != 0ull) {
        const float mn = fmaxf(m[nb], mx);
        const float corr = mn == -INFINITY ? 1.f : fast_exp2(m[nb] - mn);
        m[nb] = mn;
        l[nb] *= corr;
#pragma unroll
        for (int i = 0; i < W; ++i) oacc[nb][i] *= corr;
      }
      const float base = m[nb] == -INFINITY ? 0.f : m[nb];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float p0 = fast_exp2(x[i] - base), p1 = fast_exp2(x[i + 1] - base);
        l[nb] += p0 + p1;
        const uint32_t sc = t4.vs[i >> 1];
        // a position that the row does not see weighs nothing, whatever its scale is
        const float v0 = p0 == 0.f ? 0.f : p0 * from_bf16(sc & 0xFFFFu);
        const float v1 = p1 == 0.f ? 0.f : p1 * __builtin_bit_cast(float, sc & 0xFFFF0000u);
        uint32_t two[NP];
        split_bf16<NP>(v0, v1, two);
#pragma unroll
        for (int n = 0; n < NP; ++n) pb[nb][n][i >> 1] = two[n];
      }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const u32x4 vf = levels_bf16(t4.vw(i));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int n = 0; n < NP; ++n) oacc[nb][i] = mfma16<bf16>(vf, pb[nb][n], oacc[nb][i]);
    }
  };

  if (mine > 0) {
    Held<G> x0, x1;
    load(x0, 0, id_of(0));
    if (mine > 1) load(x1, 1, id_of(1));
    uint32_t n0 = id_of(2), n1 = id_of(3);
    for (int t = 0; t < mine; t += 2) {
      compute(x0, t);
      if (t + 2 < mine) load(x0, t + 2, n0);
      n0 = id_of(t + 4);
      if (t + 1 < mine) {
        compute(x1, t + 1);
        if (t + 3 < mine) load(x1, t + 3, n1);
        n1 = id_of(t + 5);
      }
    }
  }

  // Merge the waves.  Lane (c, g) has row rl's channels 16 i + 4 g .. + 3 for the
  // blocks i of its group.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float lt = l[nb] + __shfl_xor(l[nb], 16, 64);
    lt += __shfl_xor(lt, 32, 64);
    float *to = part[w][nb * RB + rl];
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i / 2 == grp) {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[16 * i + 4 * g + e] = oacc[nb][i][e];
      }
    if (g == 0 && grp == 0) {
      to[D] = m[nb];
      to[D + 1] = lt;
    }
  }
  __syncthreads();
  for (int i = tid; i < live_rows * (D + 2); i += 64 * NWV) {
    const int r = i / (D + 2), d = i - r * (D + 2);
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < NWV; ++v) M = fmaxf(M, part[v][r][D]);
    const float base = M == -INFINITY ? 0.f : M;
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int v = 0; v < NWV; ++v) {
      const float f = fast_exp2(part[v][r][D] - base);
      sum = fmaf(part[v][r][d], f, sum);
      total = fmaf(part[v][r][D + 1], f, total);
    }
    const int row = row0 + r;
    if (a.splits > 1) {
      a.ws[((static_cast<int64_t>(b * a.p.heads + hk) * a.splits + split) * a.rows + row) * (D + 2) + d] = d == D ? M : sum;
    } else if (d < D) {
      const int rr = row / a.len_q, qi = row - rr * a.len_q;
      static_cast<T *>(const_cast<void *>(a.o.data))[b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
                                                     qi * a.o.s2 + d] =
          static_cast<T>(total == 0.f ? 0.f : sum / total);
    }
  }
}

// One wave an output row: the splits' partial states, rescaled to their largest
// maximum.  Every lane takes the splits' (max, sum) of its share, then the wave
// walks the splits with lane d on channels d, d + 64, ...
template <typename T, int D>
__global__ __launch_bounds__(64) void attend4_merge_kernel(Attend4 a) {
  const int lane = threadIdx.x, b = blockIdx.z, hk = blockIdx.y, r = blockIdx.x;
  const int n = (a.s.len[b] + a.split - 1) / a.split;
  const float *base = a.ws + (static_cast<int64_t>(b * a.p.heads + hk) * a.splits * a.rows + r) * (D + 2);
  const int64_t stride = static_cast<int64_t>(a.rows) * (D + 2);
  constexpr int PER = (D + 63) / 64, U = 8;
  float M = -INFINITY;
  for (int s = lane; s < n; s += 64) M = fmaxf(M, base[s * stride + D]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
  const float at = M == -INFINITY ? 0.f : M;
  float acc[PER] = {}, L = 0.f;
  for (int s0 = 0; s0 < n; s0 += U) {
    float f[U], ls[U], x[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float *from = base + min(s0 + u, n - 1) * stride;
      f[u] = from[D], ls[u] = from[D + 1];
#pragma unroll
      for (int i = 0; i < PER; ++i) x[u][i] = from[min(lane + 64 * i, D - 1)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u < n) {
        const float e = fast_exp2(f[u] - at);
        L = fmaf(ls[u], e, L);
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = fmaf(x[u][i], e, acc[i]);
      }
  }
  const int rr = r / a.len_q, qi = r - rr * a.len_q;
  T *out = static_cast<T *>(const_cast<void *>(a.o.data)) + b * a.o.s0 + static_cast<int64_t>(hk * a.rep + rr) * a.o.s1 +
           qi * a.o.s2;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < D) out[lane + 64 * i] = static_cast<T>(L == 0.f ? 0.f : acc[i] / L);
}

// Column blocks of a workgroup.  Two read the cache once for twice the rows;
// their operands are more registers than fp32 queries (three parts) and 256
// channels leave.
int column_blocks(int dtype, int dim, int rows) {
  return rows > 512 / dim && dtype != TSATTN_F32 && dim < 256 ? 2 : 1;
}

}  // namespace

int attend4_split(int dtype, int dim, int heads_kv, int rows, int64_t total, int longest) {
  const int per = 512 / dim * column_blocks(dtype, dim, rows);
  const int64_t blocks = static_cast<int64_t>(heads_kv) * ((rows + per - 1) / per);
  int64_t split = total * blocks / 1024;
  split = split < 256 ? 256 : split > 4096 ? 4096 : split;
  const int64_t n = (longest + split - 1) / split;  // splits; then of equal length
  const int64_t even = n > 0 ? (longest + n - 1) / n : 0;
  return static_cast<int>((even + 127) / 128 * 128 ? (even + 127) / 128 * 128 : 128);
}

hipError_t launch_attend4(const Attend4 &a, int dtype, hipStream_t st) {
  const int dim = a.p.dim, nb = column_blocks(dtype, dim, a.rows), per = 512 / dim * nb;
  const dim3 grid(a.p.heads * ((a.rows + per - 1) / per), a.splits, a.n);
  auto launch = [&](auto t, auto g) {
    using T = decltype(t);
    constexpr int G = decltype(g)::value;
    {
      Probe pr_("attend4", st);
      if constexpr (!std::is_same_v<T, float> && G < 8) {
        if (nb == 2) attend4_kernel<T, G, 2><<<grid, dim3(64 * NWV), 0, st>>>(a);
        else attend4_kernel<T, G, 1><<<grid, dim3(64 * NWV), 0, st>>>(a);
      } else {
        attend4_kernel<T, G, 1><<<grid, dim3(64 * NWV), 0, st>>>(a);
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
