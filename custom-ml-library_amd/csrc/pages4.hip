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

template <typename T>
__device__ __forceinline__ void load8(const T *p, T (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    const u32x4 r = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e[i];
  } else {
    const f32x4 *q = reinterpret_cast<const f32x4 *>(p);
    const f32x4 a = __builtin_nontemporal_load(q), b = __builtin_nontemporal_load(q + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  }
}

// Four consecutive table entries.
template <typename T>
__device__ __forceinline__ void load4(const T *p, T (&x)[4]) {
  using V = std::conditional_t<sizeof(T) == 2, u32x2, u32x4>;
  const V r = *reinterpret_cast<const V *>(p);
  const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = e[i];
}

// A group's scale from the largest magnitude's bits (compared as integers, in
// which a NaN is the largest of all).
template <typename T>
__device__ __forceinline__ float scale_of(uint32_t m) {
  const float q = __builtin_bit_cast(float, m) / 6.f;
  uint32_t u = __builtin_bit_cast(uint32_t, q);
  u = (u + 0x1FFFFu + ((u >> 18) & 1u)) & ~0x3FFFFu;  // 5 mantissa bits
  const float s = fminf(fmaxf(__builtin_bit_cast(float, u), 0x1p-27f), most_scale<T>());
  return m >= 0x7F800000u ? __builtin_nanf("") : s;
}

// Eight codes.  The quotient comes from the reciprocal and one correction: within
// half an ulp of x / s, and exact where x / s is half way between two levels.
// For 16-bit x no other quotient comes that near to such a point (x has at most 11
// significant bits, the point times s 9), so the conversion's rounding (to nearest,
// ties to even, saturating) decides as the real quotient does.  fp32 quotients
// are truncated with a sticky last bit instead, so that none rounds onto one.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const T (&x)[8], float s) {
#pragma clang fp contract(off)
  const float rc = 1.f / s;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = static_cast<float>(x[i]);
    const float q0 = a * rc;
    q[i] = __builtin_fmaf(__builtin_fmaf(-q0, s, a), rc, q0);
    if constexpr (std::is_same_v<T, float>) {
      const float m = fabsf(q[i]), r = __builtin_fmaf(-m, s, fabsf(a));
      uint32_t u = __builtin_bit_cast(uint32_t, m);
      if (r < 0.f && u != 0u) --u;
      if (r != 0.f) u |= 1u;
      q[i] = copysignf(__builtin_bit_cast(float, u), a);
    }
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.f, 3);
  return w;
}

// One wave quantises the new positions of one tile, head and side (keys or
// values).  Lane (c, g) takes keys c and 16 + c and their channels 32 ks + 8 g .. + 7:
// 16-byte loads of which four make a group, and the words of the keys' layout.
// Values' words hold one channel of eight keys: the codes cross the wave through
// LDS.  A tile that is only partly new keeps its other positions: keys' words
// belong to one position each, values' are read, merged and written.
template <typename T, int G>
__global__ __launch_bounds__(NT) void append_kernel(RowArgs a) {
  constexpr int D = 32 * G, W = 2 * G;
  __shared__ __attribute__((aligned(16))) uint32_t lds[NW][kTile * (D / 8)];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x * NW + wv;  // (tile, side, head), the tile fastest
  const int b = blockIdx.y;
  const int hs = unit / a.tiles, ti = unit - hs * a.tiles;
  const bool values = hs & 1;
  const int h = hs >> 1;
  const int pos = a.s.len[b];
  const int tile = pos / kTile + ti, first = tile * kTile - pos;  // new position of the tile's first
  if (h >= a.p.heads || first >= a.len) return;                   // (a whole wave; no barrier follows)
  const bool full = first >= 0 && first + kTile <= a.len;
  char *to = tile4(a.p, a.s.row[b], tile, h) + (values ? 16 * D : 0);
  uint16_t *sto = reinterpret_cast<uint16_t *>(tile4(a.p, a.s.row[b], tile, h) + (values ? 34 : 32) * D);
  const View &v = values ? a.v : a.k;
  const T *src = static_cast<const T *>(v.data) + b * v.s0 + h * v.s1 + 8 * g;
  T x[2][G][8];
  bool live[2];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int t = first + 16 * kb + c;
    live[kb] = t >= 0 && t < a.len;
    const int64_t at = live[kb] ? t : (first < 0 ? 0 : first);  // (else a new position's row: in bounds)
#pragma unroll
    for (int ks = 0; ks < G; ++ks) load8<T>(src + at * v.s2 + 32 * ks, x[kb][ks]);
    if (a.cos && !values) {
#pragma unroll
      for (int ks = 0; ks < G; ++ks) {
        T cw[4], sw[4];
        const int64_t e = (pos + at) * (D / 2) + 16 * ks + 4 * g;
        load4<T>(static_cast<const T *>(a.cos) + e, cw);
        load4<T>(static_cast<const T *>(a.sin) + e, sw);
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate_pair(x[kb][ks][2 * i], x[kb][ks][2 * i + 1], cw[i], sw[i], false);
      }
    }
  }
  uint32_t word[W], sc[W];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int ks = 0; ks < G; ++ks) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        m = max(m, __builtin_bit_cast(uint32_t, static_cast<float>(x[kb][ks][i])) & 0x7FFFFFFFu);
      m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16, 64)));
      m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32, 64)));
      const float s = scale_of<T>(m);
      sc[kb * G + ks] = __builtin_bit_cast(uint32_t, s) >> 16;
      word[kb * G + ks] = codes_of<T>(x[kb][ks], s == s ? s : 1.f);
    }
  // scales: lane g stores those of words g, g + 4, ..
#pragma unroll
  for (int w0 = 0; w0 < W; w0 += 4) {
    uint32_t s = sc[w0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (w0 + i < W && g == i) s = sc[w0 + i];
    const int w = w0 + g, kb = w / G, ks = w - kb * G;
    if (w < W && (kb ? live[1] : live[0])) sto[scale4<G>(16 * kb + c, ks)] = static_cast<uint16_t>(s);
  }
  if (!values) {
    if (full) {
      if constexpr (G == 1) {
        *reinterpret_cast<u32x2 *>(to + 8 * lane) = u32x2{word[0], word[1]};
      } else {
#pragma unroll
        for (int q = 0; q < W / 4; ++q)
          *reinterpret_cast<u32x4 *>(to + (64 * q + lane) * 16) =
              u32x4{word[4 * q], word[4 * q + 1], word[4 * q + 2], word[4 * q + 3]};
      }
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (live[w / G]) *reinterpret_cast<uint32_t *>(to + word4<G>(w, lane)) = word[w];
    }
    return;
  }
  // [key][D / 2 bytes] in LDS, then each lane picks its channels' codes
  uint32_t *mine = lds[wv];
#pragma unroll
  for (int w = 0; w < W; ++w) mine[(16 * (w / G) + c) * (D / 8) + 4 * (w % G) + g] = word[w];
  wait_lgkm0();  // (own wave's writes)
  __builtin_amdgcn_sched_barrier(0);
  const uint8_t *bytes = reinterpret_cast<const uint8_t *>(mine);
  uint32_t keep = 0;  // codes of positions that are not new
  if (!full)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = first + 16 * (j >> 2) + 4 * g + (j & 3);
      if (t < 0 || t >= a.len) keep |= 0xFu << (4 * j);
    }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    uint32_t y = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = 16 * (j >> 2) + 4 * g + (j & 3);
      const uint32_t two = bytes[key * (D / 2) + 8 * w + (c >> 1)];
      y |= ((two >> (4 * (c & 1))) & 0xFu) << (4 * j);
    }
    word[w] = y;
  }
  if (keep) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      uint32_t *at = reinterpret_cast<uint32_t *>(to + word4<G>(w, lane));
      if (keep != 0xFFFFFFFFu) *at = (*at & keep) | (word[w] & ~keep);
    }
  } else if constexpr (G == 1) {
    *reinterpret_cast<u32x2 *>(to + 8 * lane) = u32x2{word[0], word[1]};
  } else {
#pragma unroll
    for (int q = 0; q < W / 4; ++q)
      *reinterpret_cast<u32x4 *>(to + (64 * q + lane) * 16) =
          u32x4{word[4 * q], word[4 * q + 1], word[4 * q + 2], word[4 * q + 3]};
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
    *reinterpret_cast<u32x4 *>(p) = u32x4{pack2<T>(y[0][0], y[0][1]), pack2<T>(y[1][0], y[1][1]),
                                          pack2<T>(y[2][0], y[2][1]), pack2<T>(y[3][0], y[3][1])};
  } else {
    reinterpret_cast<f32x4 *>(p)[0] = f32x4{y[0][0], y[0][1], y[1][0], y[1][1]};
    reinterpret_cast<f32x4 *>(p)[1] = f32x4{y[2][0], y[2][1], y[3][0], y[3][1]};
  }
}

// The values of positions first .. first + len - 1 of every sequence into k, v
// [n, heads, len, D], zero past its length.  One wave a tile, head and side;
// values' codes cross the wave through LDS as in the append.
template <typename T, int G>
__global__ __launch_bounds__(NT) void read_kernel(ReadArgs ra) {
  constexpr int D = 32 * G, W = 2 * G;
  const RowArgs &a = ra.r;
  __shared__ __attribute__((aligned(16))) uint32_t lds[NW][kTile * (D / 8)];
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
  uint32_t word[W];
  const uint16_t *sfrom = nullptr;
  const bool held = tile * kTile < n;  // (a tile past the length may have no page)
  if (held) {
    const char *base = tile4(a.p, a.s.row[b], tile, h);
    const char *from = base + (values ? 16 * D : 0);
    sfrom = reinterpret_cast<const uint16_t *>(base + (values ? 34 : 32) * D);
    if constexpr (G == 1) {
      const u32x2 r = *reinterpret_cast<const u32x2 *>(from + 8 * lane);
      word[0] = r[0], word[1] = r[1];
    } else {
#pragma unroll
      for (int q = 0; q < W / 4; ++q) {
        const u32x4 r = *reinterpret_cast<const u32x4 *>(from + (64 * q + lane) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) word[4 * q + i] = r[i];
      }
    }
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) word[w] = 0;
  }
  if (values) {
    uint32_t *mine = lds[wv];
    // words back in (q, lane) order: byte word4(w, lane)
#pragma unroll
    for (int w = 0; w < W; ++w) mine[word4<G>(w, lane) / 4] = word[w];
    wait_lgkm0();  // (own wave's writes)
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t *bytes = reinterpret_cast<const uint8_t *>(mine);
#pragma unroll
    for (int w = 0; w < W; ++w) {  // as keys' words: key 16 (w / G) + c, channels 32 (w % G) + 8 g .. + 7
      uint32_t y = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 32 * (w % G) + 8 * g + i;
        const int j = 4 * (w / G) + (c & 3);
        const uint32_t two = bytes[word4<G>(d >> 4, 16 * (c >> 2) + (d & 15)) + (j >> 1)];
        y |= ((two >> (4 * (j & 1))) & 0xFu) << (4 * i);
      }
      word[w] = y;
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int key = 16 * (w / G) + c, t = first + key;
    if (t < 0 || t >= a.len) continue;
    const float s = held ? from_bf16(sfrom[scale4<G>(key, w % G)]) : 0.f;
    store8<T>(out + static_cast<int64_t>(t) * v.s2 + 32 * (w % G) + 8 * g, word[w], s, tile * kTile + key < n);
  }
}

struct MoveArgs {
  const char *from;
  char *to;
  int64_t page_bytes;
  int32_t src[kMoves], dst[kMoves];
};

// Page blockIdx.y's share of a copy: 16 bytes a lane, four loads in flight.
__global__ __launch_bounds__(NT) void copy_kernel(MoveArgs a) {
  const u32x4 *from = reinterpret_cast<const u32x4 *>(a.from + a.src[blockIdx.y] * a.page_bytes);
  u32x4 *to = reinterpret_cast<u32x4 *>(a.to + a.dst[blockIdx.y] * a.page_bytes);
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

struct SetArgs {
  int32_t *table;
  int32_t at[kMoves], value[kMoves];
};

__global__ __launch_bounds__(512) void set_kernel(SetArgs a, int n) {
  const int i = threadIdx.x;
  if (i < n) a.table[a.at[i]] = a.value[i];
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

hipError_t launch_pages4_copy(const char *from, char *to, int64_t page_bytes, int n, const int32_t *src,
                              const int32_t *dst, hipStream_t st) {
  Probe pr_("pages4_copy", st);
  for (int i0 = 0; i0 < n; i0 += kMoves) {
    MoveArgs a{from, to, page_bytes, {}, {}};
    const int m = n - i0 < kMoves ? n - i0 : kMoves;
    for (int i = 0; i < m; ++i) a.src[i] = src[i0 + i], a.dst[i] = dst[i0 + i];
    const int64_t blocks = (page_bytes / 16 + NT * 4 - 1) / (NT * 4);
    copy_kernel<<<dim3(static_cast<unsigned>(blocks < 64 ? blocks : 64), m), dim3(NT), 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_pages4_set(int32_t *table, int n, const int32_t *at, const int32_t *value, hipStream_t st) {
  Probe pr_("pages4_set", st);
  for (int i0 = 0; i0 < n; i0 += kMoves) {
    SetArgs a{table, {}, {}};
    const int m = n - i0 < kMoves ? n - i0 : kMoves;
    for (int i = 0; i < m; ++i) a.at[i] = at[i0 + i], a.value[i] = value[i0 + i];
    static_assert(kMoves <= 512, "one lane an entry");
    set_kernel<<<dim3(1), dim3((m + 63) / 64 * 64), 0, st>>>(a, m);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tsattn
