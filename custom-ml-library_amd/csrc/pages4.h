// A key/value cache held in 4 bits, in pages: the format, and what the kernels
// over it share (pages4.hip: append, read back, page copies; attend4.hip:
// attention).
//
// Values.  Each 32 channels of a key's or value's row x share a scale
//   s = round6(max|x| / 6)   (the quotient in fp32; 6 significant bits, ties to
//   even), at least 2^-27 and at most the largest s whose 6 s the cache's dtype
//   holds; NaN when one of the 32 is not finite,
// and each channel has a code: the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (e2m1) to
// |x| / s, ties to the even code, with the sign in bit 3.  A level has 2
// significant bits, so level * s has 8: what the cache stands for is exact in
// bf16 and fp32, and in f16 down to its subnormal numbers (s >= 2^-18).  That is
// why s keeps 6 bits and not the 8 that its bf16 storage could hold: the
// coarser scale moves a code's error by under 1%, and dequantising to 16 bits
// (the prompt path, get) then rounds nothing.
//
// Layout.  A page holds `page` positions (32, 64, 128, ...) of every head; its
// heads' tiles of 32 positions follow each other, each one run of 36 D bytes:
//   keys' codes 16 D | values' codes 16 D | keys' scales 2 D | values' scales 2 D.
// Codes lie in the order in which a wave's matrix operands take them, so that a
// tile goes from memory to registers by 16-byte loads, lane after lane, and
// through no LDS.  With lane = 16 g + c and G = D / 32 groups, lane's words are
//   keys   w = kb G + ks: key 16 kb + c, channels 32 ks + 8 g .. + 7;
//   values w = 0 .. 2 G - 1: channel 16 w + c, keys 4 g .. + 3 and 16 + 4 g .. + 3,
// eight codes a word, the first in the lowest bits; words 4 q .. 4 q + 3 of a
// lane are its 16 bytes of chunk q, at (64 q + lane) 16 (D = 32: 2 words, 8 bytes,
// at 8 lane).  Scales (bf16) of key k, group s: element ((k % 16) / 4 * G + s) 8 +
// k / 16 * 4 + k % 4: the eight that a lane needs are 16 bytes.
#pragma once

#include "mfma_common.h"

namespace tsattn {

constexpr int kTile = 32;     // positions a tile
constexpr int kLongest = 1 << 27;  // positions a sequence: splits of 4096 stay within a grid's 65535
constexpr int kSeqs = 256;    // sequences a launch: their numbers travel by value
constexpr int kMoves = 240;   // page copies, and table entries, a launch (under 4 KiB of arguments)

// Sequences of a launch: row of the page table, cached positions (the kernels'
// arguments hold them, so no copy to the device precedes a launch and a captured
// launch replays what it was captured with).
struct Seqs {
  int32_t row[kSeqs], len[kSeqs];
};

struct Pages4 {
  char *pool;
  int64_t page_bytes;
  int32_t pages, heads, per_page, dim;  // a page: 2^per_page tiles of every head
  const int32_t *table;                 // [rows, stride] page numbers
  int64_t stride;
};

inline int64_t page4_bytes(int heads, int page, int dim) {
  return static_cast<int64_t>(heads) * (page / kTile) * 36 * dim;
}

// Tile `tile` of a sequence, head h, in page id.  Page numbers out of range (a table that
// its owner did not fill) read page 0 rather than memory outside the pool.
__device__ __forceinline__ char *tile4_at(const Pages4 &p, uint32_t id, int tile, int h) {
  const int64_t page = id < static_cast<uint32_t>(p.pages) ? id : 0;
  const int in = tile & ((1 << p.per_page) - 1);
  return p.pool + page * p.page_bytes + ((static_cast<int64_t>(h) << p.per_page) + in) * 36 * p.dim;
}
// The same, by table row.
__device__ __forceinline__ char *tile4(const Pages4 &p, int row, int tile, int h) {
  const uint32_t id = static_cast<uint32_t>(p.table[row * p.stride + (tile >> p.per_page)]);
  return tile4_at(p, id, tile, h);
}

// Byte of word w of a lane's codes.
template <int G>
__device__ __forceinline__ constexpr int word4(int w, int lane) {
  return G == 1 ? lane * 8 + w * 4 : ((w >> 2) * 64 + lane) * 16 + (w & 3) * 4;
}
// Element of the scale of key k, group s.
template <int G>
__device__ __forceinline__ constexpr int scale4(int k, int s) {
  return (((k & 15) >> 2) * G + s) * 8 + (k >> 4) * 4 + (k & 3);
}

__device__ __forceinline__ float from_bf16(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }

// Eight codes as eight bf16 levels (exact), and as floats.
__device__ __forceinline__ u32x4 levels_bf16(uint32_t w) {
  u32x4 y;
  y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0));
  y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1));
  y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2));
  y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3));
  return y;
}

hipError_t launch_pages4_append(const Pages4 &p, int dtype, int n, int len, View k, View v, const Seqs &s,
                                const void *cos, const void *sin, hipStream_t st);
hipError_t launch_pages4_read(const Pages4 &p, int dtype, int n, int len, View k, View v, const Seqs &s,
                              const int32_t *first, hipStream_t st);
hipError_t launch_pages4_apply(const char *from, char *to, int64_t page_bytes, int moves, const int32_t *src,
                               const int32_t *dst, int32_t *table, int sets, const int32_t *at,
                               const int32_t *value, hipStream_t st);

// pages4_table.hip
int32_t pages4_grow(tsattn_pages4_host *h, int32_t n, const int32_t *rows, int32_t steps, int32_t *src,
                    int32_t *dst, int32_t *copies);
void pages4_cut(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *lengths);
void pages4_reorder(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *index, int32_t *old);
int32_t pages4_clone(const tsattn_pages4_host *from, int32_t n, const int32_t *rows, tsattn_pages4_host *to,
                     int32_t *number, int32_t *src, int32_t *dst);
int32_t pages4_compact(tsattn_pages4_host *h, int32_t *number, int32_t *src, int32_t *dst, int32_t *copies);
int32_t pages4_changes(const tsattn_pages4_host *h, int32_t *at, int32_t *value);
void pages4_sent(tsattn_pages4_host *h, int32_t sets, const int32_t *at, const int32_t *value);

// Attention of len_q queries a sequence (q, out: [n, heads_q, len_q, dim]) over
// the cached positions, the queries' own the last len_q of them.
struct Attend4 {
  Pages4 p;
  View q, o;
  float *ws;
  const void *cos, *sin;  // rotate the queries; or NULL
  int n, rep, len_q, first, rows, causal;  // rows: of a KV head, rep len_q in all, from the launch's first
  int split, splits;      // positions a split (a multiple of 32), splits of the longest sequence
  int wide;                    // whether a column is a row, not a group of one
  int columns, waves, blocks;  // column blocks (1 or 2) and waves of a workgroup; workgroups a KV head's rows take
  float sl, sign;         // |scale| * log2(e) and the scale's sign, with the queries; 1 and 0 for no scale
  FastDiv by_len_q;
  Seqs s;
};
// Fills split, splits, columns, waves and blocks in for the sequences' lengths.
void plan_attend4(Attend4 *a, int dtype, const int32_t *lens);
hipError_t launch_attend4(const Attend4 &a, int dtype, hipStream_t st);

}  // namespace tsattn
