// Log probabilities of given tokens, the entropy of their rows and the rows' most
// likely tokens, with the VJP.  No counterpart in the reference, whose cross entropy
// (src/tensorsmith/nn/functional.py:397-472) keeps the whole log-softmax.
//
// With m = max z, l = sum_j exp(z_j - m) over a row z of V logits:
//   log p_y = (z_y - m) - ln l,   H = ln l - (1 / l) sum_j exp(z_j - m) (z_j - m),
// where both terms of H are >= 0, so that nothing cancels; a logit of -inf adds
// nothing.  The VJP, for upstream gradients g of log p_y, gh of H and t_i of the top
// tokens' log probabilities (at indices k_i), G = g + sum_i t_i:
//   dz_j = -p_j (G + gh (ln p_j + H)) + [j = y] g + sum_i [j = k_i] t_i,
// p_j from z_j - m, which does not overflow upwards, and the log2 l that the forward kept.
//
// A lane's sums are in log2 units, t_j = z_j log2 e - b as one fused operation, b = m log2 e
// as it rounds.  What that rounding takes, r = m log2 e - b, is in every t of the lane alike,
// and `exact` takes it out again before sums meet, as 2^-r.  That needs an r that exp2 can
// hold: a largest logit whose b is past kFar (2^20, r at most 2^-5), such as a mask of -1e10
// or of the type's lowest value, whose product with log2 e may overflow besides, turns the
// wave to t_j = (z_j - m) log2 e from then on, two instructions a logit more.  (For every
// logit of every row they would cost a tenth of the forward: 116 -> 128 us.)
//
// Bound by HBM: the forward reads the logits once, the VJP reads them and writes the
// gradient.  One pass in each: a lane keeps a running (m, l, sum 2^t t) and rescales it
// once for every four 16-byte pieces.  The forward is about as far from the vector units'
// bound: 6 instructions a logit; 11 of them (selects for rows' ends and -inf on every
// one) took 131 us where 8192 rows of 50021 bf16, a fifth of them ignored, take 108
// (6.1 TB/s).  The VJP of those takes 285 us, 5.2 TB/s of reads and writes, as a copy; 331
// before its rows' pieces began on whole lines of memory.
//
// A row belongs to one wave (wave_rows), to a workgroup of four, or, when the rows
// are too few to fill the chip, to several workgroups that each take a part of it; a
// second kernel then combines the parts in their order.  Results depend on the sizes
// alone, no atomics.
//
// The top tokens: each wave keeps the 64 best (logit, index) pairs it saw, sorted, one
// a lane, as 64-bit keys whose order is the logits' with ties to the lower index, and a
// threshold, the top-th best of them.  A piece whose largest logit is not above the
// threshold, which is nearly every one, costs a comparison; keys above it go to a
// buffer in LDS, 64 of which are sorted and merged at a time.  The first piece would
// send every element there: when many lanes have candidates, the top-th best of the
// lanes' own best becomes the threshold first (top elements at least are as good).
#include <type_traits>

#include "tsattn_internal.h"

namespace tsattn {
namespace {

constexpr int NT = 256;
constexpr int NW = NT / 64;
constexpr int U = 4;         // 16-byte pieces a lane has in flight
constexpr int PENDING = 64 + 64 * 8;  // keys a wave's buffer holds: < 64 left over, and one piece of each lane
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = 1048576.f;  // b from which on z log2 e - b is not taken
constexpr float kLeast = -1e4f;    // 2^t is 0 from here on, and so is its product with t and a factor below 3e34

struct ProbArgs {
  int64_t rows;
  int vocab, top, splits;
  const void *z;
  int64_t zs;  // row stride in elements
  const void *tokens;
  int token_bytes;
  int64_t ignore;
  float *logp, *entropy, *stats;  // stats: [rows][2] = m, log2 l
  float *top_logp;
  int64_t *top_index;
  float *part;                   // [rows][splits][4]: m, l, sum 2^t t
  unsigned long long *part_top;  // [rows][splits][top]
  // VJP
  const float *g, *gh, *gt, *saved_entropy;
  const int64_t *saved_index;
  void *dz;
};

typedef unsigned long long u64;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
constexpr int kVE = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(u32x4 raw, float (&x)[kVE<T>]) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned bits = raw[e];  // (a bit cast of raw[e] itself takes the vector's first element)
      x[e] = __builtin_bit_cast(float, bits);
    }
  } else if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned bits = (e & 1) ? raw[e >> 1] & 0xFFFF0000u : raw[e >> 1] << 16;
      x[e] = __builtin_bit_cast(float, bits);
    }
  } else {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 h = __builtin_bit_cast(h8, raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(h[e]);
  }
}

__device__ __forceinline__ int64_t token_of(const ProbArgs &a, int64_t row) {
  return a.token_bytes == 8 ? static_cast<const int64_t *>(a.tokens)[row]
                            : static_cast<const int32_t *>(a.tokens)[row];
}

// ---------------------------------------------------------------------------
// Running sums: m the largest logit, l = sum 2^t, w = sum 2^t t.
// ---------------------------------------------------------------------------
struct Sums {
  float m, l, w;
};

// (a base that keeps 2^(-inf - base) = 0 while nothing but -inf has come)
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
// b, rounded here (a fused operation further on would round it otherwise)
__device__ __forceinline__ float scaled(float m) {
  float b = base_of(m) * kLog2e;
  asm("" : "+v"(b));
  return b;
}

__device__ __forceinline__ void shift(Sums &s, float d) {
  const float c = __builtin_amdgcn_exp2f(d);
  // an empty sum stays empty whatever the bases (0 * inf is NaN)
  s.w = s.l == 0.f ? s.w : c * fmaf(s.l, fmaxf(d, kLeast), s.w);
  s.l = s.l == 0.f ? s.l : s.l * c;
}
// Sums over t = (z - m) log2 e, to another m.
__device__ __forceinline__ void rebase(Sums &s, float m) {
  shift(s, (s.m - m) * kLog2e);
  s.m = m;
}
// Sums over t = z log2 e - b as sums over (z - m) log2 e.
__device__ __forceinline__ Sums exact(Sums s, float b) {
  const float r = fmaf(base_of(s.m), kLog2e, -b), c = __builtin_amdgcn_exp2f(-r);
  return Sums{s.m, s.l * c, fmaf(-r, s.l, s.w) * c};
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  return Sums{m, a.l + b.l, a.w + b.w};
}
__device__ __forceinline__ Sums wave_join(Sums s) {
  float m = s.m;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  rebase(s, m);
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    s.l += __shfl_xor(s.l, k, 64);
    s.w += __shfl_xor(s.w, k, 64);
  }
  return s;
}

// The largest of N values that is not a NaN (two an instruction, where fmaxf would also
// canonicalise each; a NaN shows in the sums).
template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int e = 1; e + 1 < N; e += 2) asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[e]), "v"(x[e + 1]));
  if constexpr (N % 2 == 0) asm("v_max_f32 %0, %1, %2" : "=v"(m) : "v"(m), "v"(x[N - 1]));
  return m;
}

// Adds N logits, none above m; `own` becomes their sum of exponentials (NaN where one is
// NaN or +inf).  NEAR: z log2 e - base, where a logit of -inf makes w a NaN (0 times -inf);
// SAFE: the same, but that, at an instruction a logit; FAR: (z - base) log2 e, as safe.
enum Sort { NEAR, SAFE, FAR };
template <Sort S, int N>
__device__ __forceinline__ void add(Sums &s, const float (&x)[N], float base, float &own) {
  float l = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float t = S == FAR ? (x[e] - base) * kLog2e : fmaf(x[e], kLog2e, -base);
    const float p = __builtin_amdgcn_exp2f(t);
    l += p;
    s.w = fmaf(p, S == NEAR ? t : fmaxf(t, kLeast), s.w);
  }
  s.l += l;
  own = l;
}

// ---------------------------------------------------------------------------
// The best keys.
// ---------------------------------------------------------------------------
// Keys order as (logit, lower index first); a NaN is the largest, -0 equals 0.
__device__ __forceinline__ u64 key_of(float z, unsigned index) {
  unsigned u = __builtin_bit_cast(unsigned, z + 0.f);
  u = z != z ? 0x7FFFFFFFu : u;
  u ^= (u >> 31) ? 0xFFFFFFFFu : 0x80000000u;
  return static_cast<u64>(u) << 32 | ~index;
}
__device__ __forceinline__ float key_logit(u64 key) {
  const unsigned u = static_cast<unsigned>(key >> 32);
  return __builtin_bit_cast(float, (u >> 31) ? u ^ 0x80000000u : ~u);
}
// The value of lane l ^ STRIDE, without LDS: data-parallel moves inside a row of 16,
// v_permlane16_swap / 32_swap (the odd rows or half of one register for the even of
// another) between them.
template <int STRIDE>
__device__ __forceinline__ unsigned of_lane_xor(unsigned x, int lane) {
  if constexpr (STRIDE == 1) return __builtin_amdgcn_update_dpp(x, x, 0xB1, 0xF, 0xF, false);
  else if constexpr (STRIDE == 2) return __builtin_amdgcn_update_dpp(x, x, 0x4E, 0xF, 0xF, false);
  else if constexpr (STRIDE == 4) {
    const unsigned y = __builtin_amdgcn_update_dpp(x, x, 0x104, 0xF, 0x5, false);  // row_shl:4 into the lower of each 8
    return __builtin_amdgcn_update_dpp(y, x, 0x114, 0xF, 0xA, false);              // row_shr:4 into the upper
  } else if constexpr (STRIDE == 8) {
    return __builtin_amdgcn_update_dpp(x, x, 0x128, 0xF, 0xF, false);  // row_ror:8
  } else {
    unsigned a = x, b = x;
    if constexpr (STRIDE == 16) asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    else asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return lane & STRIDE ? a : b;
  }
}
// One exchange of a bitonic network: lanes l and l ^ STRIDE, the larger to the lower
// lane where `down`.
template <int STRIDE>
__device__ __forceinline__ u64 exchange(u64 x, int lane, bool down) {
  const unsigned lo = of_lane_xor<STRIDE>(static_cast<unsigned>(x), lane);
  const unsigned hi = of_lane_xor<STRIDE>(static_cast<unsigned>(x >> 32), lane);
  const u64 y = static_cast<u64>(hi) << 32 | lo;
  return (((lane & STRIDE) == 0) == down) == (x > y) ? x : y;
}
template <int STRIDE>
__device__ __forceinline__ u64 ripple(u64 x, int lane, bool down) {
  x = exchange<STRIDE>(x, lane, down);
  if constexpr (STRIDE > 1) x = ripple<STRIDE / 2>(x, lane, down);
  return x;
}
template <int SIZE = 2>
__device__ __forceinline__ u64 sort_up(u64 x, int lane) {
  x = ripple<SIZE / 2>(x, lane, (lane & SIZE) != 0);
  if constexpr (SIZE < 64) x = sort_up<SIZE * 2>(x, lane);
  return x;
}
// The 64 best, falling, of a list that falls and one that rises.
__device__ __forceinline__ u64 merge_down(u64 best, u64 rising, int lane) {
  return ripple<32>(best > rising ? best : rising, lane, true);
}
// A lane's value in scalar registers.
__device__ __forceinline__ u64 of_lane(u64 x, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<unsigned>(x), lane);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<unsigned>(x >> 32), lane);
  return static_cast<u64>(hi) << 32 | lo;
}

struct Best {
  u64 best = 0;       // this lane's rank of the wave's list; 0: none
  u64 least = 0;      // keys must be above it (0: all are)
  float least_z = 0;  // its logit
  int pending = 0;
  u64 *buffer;

  __device__ __forceinline__ void raise(u64 key) {
    if (key > least) {
      least = key;
      least_z = key_logit(least);
    }
  }
  __device__ __forceinline__ void take(int n, int top, int lane) {
    // the buffer's last n <= 64 keys (other lanes wrote them)
    pending -= n;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u64 key = lane < n ? buffer[pending + lane] : 0;
    best = merge_down(best, sort_up(key, lane), lane);
    raise(of_lane(best, top - 1));
  }
  // N logits a lane from `index` on, n of them there; call in step, indexes rising.
  template <int N>
  __device__ __forceinline__ void offer(const float (&x)[N], float mx, float own, unsigned index, int n, int top,
                                        int lane) {
    const bool maybe = n > 0 && (least == 0 || !(mx <= least_z) || own != own);
    const u64 lanes = __ballot(maybe);
    if (lanes == 0) return;
    const int count = __popcll(lanes);
    if (count > top && count > 24) {
      u64 key = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const u64 k = e < n ? key_of(x[e], index + e) : 0;
        key = k > key ? k : key;
      }
      key = of_lane(sort_up(key, lane), 64 - top);
      if (key) raise(key - 1);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const u64 key = e < n ? key_of(x[e], index + e) : 0;
      const u64 pass = __ballot(key > least);
      if (pass == 0) continue;
      if (key > least) buffer[pending + __popcll(pass & ((u64(1) << lane) - 1))] = key;
      pending += __popcll(pass);
    }
    while (pending >= 64) take(64, top, lane);
  }
  __device__ __forceinline__ void finish(int top, int lane) {
    if (pending) take(pending, top, lane);
  }
};

// ---------------------------------------------------------------------------
// Forward.
// ---------------------------------------------------------------------------
// What a row's sums (and with TOP its best keys, one a lane) say; one wave.
template <typename T, bool TOP>
__device__ __forceinline__ void results(const ProbArgs &a, int64_t row, Sums s, u64 best, int lane) {
  // (all logits -inf: l = 0; log p is NaN as -inf - -inf is)
  const float m = s.m, log2l = log2f(s.l);
  if (lane == 0) {
    const int64_t y = token_of(a, row);
    const float z = y >= 0 && y < a.vocab ? static_cast<float>(static_cast<const T *>(a.z)[row * a.zs + y]) : NAN;
    a.logp[row] = fmaf(-log2l, kLn2, z - m);
    a.entropy[row] = m == -INFINITY ? NAN : (log2l - s.w / s.l) * kLn2;
    if (a.stats) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = log2l;
    }
  }
  if constexpr (TOP) {
    if (lane < a.top) {
      a.top_logp[row * a.top + lane] = fmaf(-log2l, kLn2, key_logit(best) - m);
      a.top_index[row * a.top + lane] = ~static_cast<unsigned>(best);
    }
  }
}

__device__ __forceinline__ void ignored(const ProbArgs &a, int64_t row, int lane, bool top) {
  if (lane == 0) {
    a.logp[row] = 0.f;
    a.entropy[row] = 0.f;
    if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.f;
  }
  if (top && lane < a.top) {
    a.top_logp[row * a.top + lane] = -INFINITY;
    a.top_index[row * a.top + lane] = -1;
  }
}

// A row as 16-byte pieces: `head` elements (at most 63) up to the first whole 128-byte
// line, so that no two waves share a line, `pieces`, then what is left.
template <typename T>
struct Row {
  const T *z;
  int head, pieces, tail;
  __device__ __forceinline__ Row(const T *p, int vocab) : z(p) {
    const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) & 127u);
    head = min(vocab, static_cast<int>((128u - off) % 128u / sizeof(T)));
    pieces = (vocab - head) / kVE<T>;
    tail = vocab - head - pieces * kVE<T>;
  }
};

// WPR: waves a row has in the workgroup, 1 or NW.
template <typename T, int WPR, bool TOP>
__global__ __launch_bounds__(NT) void probs_kernel(ProbArgs a) {
  constexpr int VE = kVE<T>, LANES = WPR * 64;
  __shared__ u64 buffers[TOP ? NW * PENDING : 1];
  __shared__ float red[NW][4];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (NW / WPR) + (WPR == 1 ? w : 0);
  const int64_t row = WPR == 1 ? id : id / a.splits;
  const int part = WPR == 1 ? 0 : static_cast<int>(id % a.splits);
  if (row >= a.rows) return;  // (WPR = NW: of the whole workgroup, and no barrier follows for WPR = 1)
  if (token_of(a, row) == a.ignore) {
    if (part == 0 && (WPR == 1 || w == 0)) ignored(a, row, lane, TOP);
    return;
  }
  const Row<T> r(static_cast<const T *>(a.z) + row * a.zs, a.vocab);
  const int splits = WPR == 1 ? 1 : a.splits;
  const int p0 = static_cast<int>(static_cast<int64_t>(r.pieces) * part / splits);
  const int p1 = static_cast<int>(static_cast<int64_t>(r.pieces) * (part + 1) / splits);
  Sums s{-INFINITY, 0.f, 0.f};
  Best top;
  top.buffer = buffers + (TOP ? w * PENDING : 0);
  bool far = false;  // of the wave: its sums are over (z - m) log2 e
  float base = 0.f;  // b, or far m
  auto raise = [&](float most) __attribute__((always_inline)) {
    if (!far) {
      const float b = scaled(most);
      if (__ballot(fabsf(b) > kFar) == 0ull) {
        shift(s, base - b);
        s.m = most;
        base = b;
        return;
      }
      s = exact(s, base);
      far = true;
    }
    rebase(s, most);
    base = base_of(most);
  };
  // the elements in front of the first piece, one a lane
  auto single = [&](int first, int n) {
    const float x[1] = {lane < n ? static_cast<float>(r.z[first + lane]) : -INFINITY};
    float own;
    raise(fmaxf(s.m, x[0]));
    if (far) add<FAR>(s, x, base, own);
    else add<SAFE>(s, x, base, own);
    if constexpr (TOP) top.offer(x, x[0], own, first + lane, lane < n ? 1 : 0, a.top, lane);
  };
  const int l0 = (WPR == 1 ? 0 : w * 64) + lane;
  if (part == 0 && (WPR == 1 || w == 0) && r.head) single(0, r.head);
  const u32x4 *pieces = reinterpret_cast<const u32x4 *>(r.z + r.head);
  // U pieces a lane ahead of those it works on
  u32x4 raw[U], next[U];
  auto load = [&](int i, u32x4 (&x)[U]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * LANES + l0;
      if (at < p1) x[u] = __builtin_nontemporal_load(pieces + at);
    }
  };
  load(p0, raw);
  for (int i = p0; i < p1; i += LANES * U) {
    load(i + LANES * U, next);
    float x[U][VE], mx[U], most = s.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * LANES >= p1) break;
      unpack<T>(raw[u], x[u]);
      // (the whole workgroup's test first: selects on every piece are an instruction an element)
      if (i + (u + 1) * LANES > p1 && i + u * LANES + l0 >= p1) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[u][e] = -INFINITY;
      }
      mx[u] = largest(x[u]);
      most = fmaxf(most, mx[u]);
    }
    raise(most);
    const Sums before = s;
    float own[U];
    if (far) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * LANES >= p1) break;
        add<FAR>(s, x[u], base, own[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * LANES >= p1) break;
        add<NEAR>(s, x[u], base, own[u]);
      }
      if (__ballot(s.w != s.w) != 0ull) {  // a logit of -inf: again
        s = before;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i + u * LANES >= p1) break;
          add<SAFE>(s, x[u], base, own[u]);
        }
      }
    }
    if constexpr (TOP) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * LANES >= p1) break;
        const int at = i + u * LANES + l0;
        top.offer(x[u], mx[u], own[u], r.head + at * VE, at < p1 ? VE : 0, a.top, lane);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
  }
  if (part == splits - 1 && (WPR == 1 || w == NW - 1) && r.tail) single(a.vocab - r.tail, r.tail);
  s = wave_join(far ? s : exact(s, base));
  if constexpr (TOP) top.finish(a.top, lane);
  if constexpr (WPR > 1) {
    if (lane == 0) red[w][0] = s.m, red[w][1] = s.l, red[w][2] = s.w;
    if constexpr (TOP) top.buffer[63 - lane] = top.best;  // (rising, as merge_down takes it)
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < NW; ++k) {
      s = join(s, Sums{red[k][0], red[k][1], red[k][2]});
      if constexpr (TOP) top.best = merge_down(top.best, buffers[k * PENDING + lane], lane);
    }
    if (splits > 1) {
      if (lane == 0) {
        float *p = a.part + 4 * id;
        p[0] = s.m, p[1] = s.l, p[2] = s.w;
      }
      if constexpr (TOP)
        if (lane < a.top) a.part_top[id * a.top + lane] = top.best;
      return;
    }
  }
  results<T, TOP>(a, row, s, top.best, lane);
}

// The parts of a row; a workgroup a row, whose waves share the parts' top keys (in any
// order: the keys are all different).
template <typename T, bool TOP>
__global__ __launch_bounds__(NT) void probs_merge_kernel(ProbArgs a) {
  __shared__ u64 lists[TOP ? NW * 64 : 1];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  if (token_of(a, row) == a.ignore) return;
  u64 best = 0;
  if constexpr (TOP) {
    const u64 *keys = a.part_top + row * a.splits * a.top;
    for (int i = w; i < a.splits; i += 4 * NW) {
      u64 more[4];  // four loads in flight
#pragma unroll
      for (int u = 0; u < 4; ++u)
        more[u] = i + u * NW < a.splits && 63 - lane < a.top ? keys[(i + u * NW) * a.top + 63 - lane] : 0;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * NW < a.splits) best = merge_down(best, more[u], lane);
    }
    lists[w * 64 + 63 - lane] = best;
    __syncthreads();
  }
  if (w) return;
  if constexpr (TOP) {
#pragma unroll
    for (int k = 1; k < NW; ++k) best = merge_down(best, lists[k * 64 + lane], lane);
  }
  // (lane i starts with part i; more parts than lanes do not occur, kMaxSplits)
  Sums s{-INFINITY, 0.f, 0.f};
  if (lane < a.splits) {
    const float *p = a.part + 4 * (row * a.splits + lane);
    s = Sums{p[0], p[1], p[2]};
  }
  results<T, TOP>(a, row, wave_join(s), best, lane);
}

// ---------------------------------------------------------------------------
// VJP.
// ---------------------------------------------------------------------------
template <typename T, int N>
__device__ __forceinline__ void store_piece(T *p, const float (&x)[N]) {
  typedef T V __attribute__((ext_vector_type(N)));
  V y;
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = static_cast<T>(x[e]);
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), reinterpret_cast<u32x4 *>(p));
}

// A workgroup takes part `part` of a row (WPR = NW), or each wave a row.  The gradient
// is contiguous: its rows start where they may, so its pieces are the gradient's own
// (the logits' are read by element where the two do not lie alike).
template <typename T, int WPR, bool TOP>
__global__ __launch_bounds__(NT) void probs_vjp_kernel(ProbArgs a) {
  constexpr int VE = kVE<T>, LANES = WPR * 64;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (NW / WPR) + (WPR == 1 ? w : 0);
  const int splits = WPR == 1 ? 1 : a.splits;
  const int64_t row = id / splits;
  const int part = static_cast<int>(id % splits);
  if (row >= a.rows) return;
  const T *z = static_cast<const T *>(a.z) + row * a.zs;
  T *dz = static_cast<T *>(a.dz) + row * a.vocab;
  const Row<T> r(dz, a.vocab);
  const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u) == 0;
  const int p0 = static_cast<int>(static_cast<int64_t>(r.pieces) * part / splits);
  const int p1 = static_cast<int>(static_cast<int64_t>(r.pieces) * (part + 1) / splits);
  const int l0 = (WPR == 1 ? 0 : w * 64) + lane;
  const bool has_head = part == 0 && (WPR == 1 || w == 0), has_tail = part == splits - 1 && (WPR == 1 || w == NW - 1);
  const int64_t y = token_of(a, row);
  if (y == a.ignore) {
    const float none[VE] = {};
    if (has_head && lane < r.head) dz[lane] = static_cast<T>(0.f);
    for (int i = p0 + l0; i < p1; i += LANES) store_piece(dz + r.head + i * VE, none);
    if (has_tail && lane < r.tail) dz[a.vocab - r.tail + lane] = static_cast<T>(0.f);
    return;
  }
  const float m = a.stats[2 * row], log2l = a.stats[2 * row + 1];
  float g = a.g ? a.g[row] : 0.f;
  if (y < 0 || y >= a.vocab) g = a.g ? NAN : 0.f;  // (its log probability is NaN)
  const float gh = a.gh ? a.gh[row] : 0.f;
  float all = g;
  if constexpr (TOP)
    for (int i = 0; i < a.top; ++i) all += a.gt[row * a.top + i];
  const float c = gh == 0.f ? all : fmaf(gh, a.saved_entropy[row], all);
  const float gl = gh * kLn2;
  auto at_logit = [&](float x) {
    const float t = fmaf(x - m, kLog2e, -log2l);  // log2 p
    return -__builtin_amdgcn_exp2f(t) * fmaf(gl, fmaxf(t, kLeast), c);
  };
  const int yi = y >= 0 && y < a.vocab ? static_cast<int>(y) : -1;
  auto single = [&](int j) {
    const float d = at_logit(static_cast<float>(z[j]));
    dz[j] = static_cast<T>(j == yi ? d + g : d);
  };
  if (has_head && lane < r.head) single(lane);
  u32x4 raw[U], next[U];
  auto load = [&](int i, u32x4 (&x)[U]) __attribute__((always_inline)) {
    if (alike) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * LANES < p1)
          x[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(z + r.head) + i + u * LANES);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * LANES < p1) {
          typedef T V __attribute__((ext_vector_type(VE)));
          V v;
          const T *from = z + r.head + (i + u * LANES) * VE;
#pragma unroll
          for (int e = 0; e < VE; ++e) v[e] = from[e];
          x[u] = __builtin_bit_cast(u32x4, v);
        }
    }
  };
  load(p0 + l0, raw);
  for (int i = p0 + l0; i < p1; i += LANES * U) {
    load(i + LANES * U, next);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * LANES;
      if (at >= p1) break;
      float x[VE];
      unpack<T>(raw[u], x);
      const int j0 = r.head + at * VE;
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = at_logit(x[e]);
      if (static_cast<unsigned>(yi - j0) < static_cast<unsigned>(VE)) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] += e == yi - j0 ? g : 0.f;
      }
      store_piece(dz + j0, x);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
  }
  if (has_tail && lane < r.tail) single(a.vocab - r.tail + lane);
  if constexpr (TOP) {
    // the top tokens' elements again, whole, once the part's others are written
    __threadfence();
    if constexpr (WPR > 1) __syncthreads();
    const int first = part == 0 ? 0 : r.head + p0 * VE, last = part == splits - 1 ? a.vocab : r.head + p1 * VE;
    if (l0 < a.top) {
      const int64_t j = a.saved_index[row * a.top + l0];
      if (j >= first && j < last) {
        float d = at_logit(static_cast<float>(z[j])) + a.gt[row * a.top + l0];
        if (j == yi) d += g;
        dz[j] = static_cast<T>(d);
      }
    }
  }
}

constexpr int kMaxSplits = 64;

// Rows short enough for a wave each: four of them cost the workgroup's reduction between
// its waves (8192 rows of 2000 bf16, forward and VJP: 14 and 15 us, a workgroup a row 21
// and 23; of 4000: 18 and 26, against 25 and 28; of 8000 the VJP is slower, 52 and 46).
// Few rows have the chip to themselves and gain from four waves sooner (64 rows of 3500,
// five top tokens: 15 us a wave a row, 11 a workgroup; of 1500: 11 both).
bool wave_rows(int64_t rows, int vocab) { return vocab <= (rows >= 4096 ? 4096 : 2048); }

// Parts of a row: as many as give the chip's 256 CUs 4 workgroups each (64 rows of 50000
// in 1 to 16 parts: 11 us all; 256 rows, forward and VJP: 14 and 17 us in one part, 14 and
// 13 in four, 16 and 14 in eight), of 2048 logits or more (a row of 32000 with five top
// tokens: 14.4 us, with 8192 or more 16.4, with 16384 21).
int prob_splits(int64_t rows, int vocab) {
  if (wave_rows(rows, vocab)) return 1;
  int64_t s = 1024 / rows;
  if (s > vocab / 2048) s = vocab / 2048;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : static_cast<int>(s);
}

// The rows from `first` on, `rows` of them (rows in parts come in one piece, first = 0).
template <typename T>
ProbArgs some_rows(ProbArgs a, int64_t first, int64_t rows) {
  auto from = [first](auto *p, int64_t each) { return p ? p + first * each : p; };
  a.rows = rows;
  a.z = from(static_cast<const T *>(a.z), a.zs);
  a.tokens = from(static_cast<const char *>(a.tokens), a.token_bytes);
  a.logp = from(a.logp, 1), a.entropy = from(a.entropy, 1), a.stats = from(a.stats, 2);
  a.top_logp = from(a.top_logp, a.top), a.top_index = from(a.top_index, a.top);
  a.g = from(a.g, 1), a.gh = from(a.gh, 1), a.gt = from(a.gt, a.top);
  a.saved_entropy = from(a.saved_entropy, 1), a.saved_index = from(a.saved_index, a.top);
  a.dz = from(static_cast<T *>(a.dz), a.vocab);
  return a;
}

// A grid has fewer than 2^32 work-items: 2^23 workgroups at a time.
constexpr int64_t kMostGroups = int64_t(1) << 23;

template <typename T, bool TOP>
void forward(const ProbArgs &all, hipStream_t st) {
  const bool wave = wave_rows(all.rows, all.vocab);
  const int64_t most = kMostGroups * (wave ? NW : 1);
  for (int64_t first = 0; first < all.rows; first += most) {
    const ProbArgs a = some_rows<T>(all, first, all.rows - first < most ? all.rows - first : most);
    if (wave) probs_kernel<T, 1, TOP><<<dim3(static_cast<unsigned>((a.rows + NW - 1) / NW)), dim3(NT), 0, st>>>(a);
    else probs_kernel<T, NW, TOP><<<dim3(static_cast<unsigned>(a.rows * a.splits)), dim3(NT), 0, st>>>(a);
    if (a.splits > 1) probs_merge_kernel<T, TOP><<<dim3(static_cast<unsigned>(a.rows)), dim3(NT), 0, st>>>(a);
  }
}

template <typename T, bool TOP>
void backward(const ProbArgs &all, hipStream_t st) {
  const bool wave = wave_rows(all.rows, all.vocab);
  const int64_t most = kMostGroups * (wave ? NW : 1);
  for (int64_t first = 0; first < all.rows; first += most) {
    const ProbArgs a = some_rows<T>(all, first, all.rows - first < most ? all.rows - first : most);
    if (wave) probs_vjp_kernel<T, 1, TOP><<<dim3(static_cast<unsigned>((a.rows + NW - 1) / NW)), dim3(NT), 0, st>>>(a);
    else probs_vjp_kernel<T, NW, TOP><<<dim3(static_cast<unsigned>(a.rows * a.splits)), dim3(NT), 0, st>>>(a);
  }
}

}  // namespace

size_t token_probs_workspace(int64_t rows, int vocab, int top) {
  const int s = prob_splits(rows, vocab);
  return s < 2 ? 0 : static_cast<size_t>(rows) * s * (4 * sizeof(float) + top * sizeof(unsigned long long));
}

hipError_t launch_token_probs(int dtype, int64_t rows, int vocab, const void *z, int64_t zs, const void *tokens,
                              int token_bytes, int64_t ignore, int top, float *logp, float *entropy, float *stats,
                              float *top_logp, int64_t *top_index, void *ws, hipStream_t st) {
  ProbArgs a{};
  a.rows = rows, a.vocab = vocab, a.top = top, a.splits = prob_splits(rows, vocab);
  a.z = z, a.zs = zs, a.tokens = tokens, a.token_bytes = token_bytes, a.ignore = ignore;
  a.logp = logp, a.entropy = entropy, a.stats = stats, a.top_logp = top_logp, a.top_index = top_index;
  a.part_top = static_cast<unsigned long long *>(ws);
  a.part = reinterpret_cast<float *>(a.part_top + (a.splits > 1 ? rows * a.splits * top : 0));
  Probe pr_("token_probs", st);
  if (dtype == TSATTN_F32) top ? forward<float, true>(a, st) : forward<float, false>(a, st);
  else if (dtype == TSATTN_F16) top ? forward<f16, true>(a, st) : forward<f16, false>(a, st);
  else top ? forward<bf16, true>(a, st) : forward<bf16, false>(a, st);
  return hipGetLastError();
}

hipError_t launch_token_probs_backward(int dtype, int64_t rows, int vocab, const void *z, int64_t zs,
                                       const void *tokens, int token_bytes, int64_t ignore, int top,
                                       const float *stats, const float *entropy, const int64_t *top_index,
                                       const float *g, const float *gh, const float *gt, void *dz, hipStream_t st) {
  ProbArgs a{};
  a.rows = rows, a.vocab = vocab, a.top = top, a.splits = prob_splits(rows, vocab);
  a.z = z, a.zs = zs, a.tokens = tokens, a.token_bytes = token_bytes, a.ignore = ignore;
  a.stats = const_cast<float *>(stats), a.saved_entropy = entropy, a.saved_index = top_index;
  a.g = g, a.gh = gh, a.gt = gt, a.dz = dz;
  Probe pr_("token_probs_backward", st);
  if (dtype == TSATTN_F32) gt ? backward<float, true>(a, st) : backward<float, false>(a, st);
  else if (dtype == TSATTN_F16) gt ? backward<f16, true>(a, st) : backward<f16, false>(a, st);
  else gt ? backward<bf16, true>(a, st) : backward<bf16, false>(a, st);
  return hipGetLastError();
}

}  // namespace tsattn
