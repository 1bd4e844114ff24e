// Matrix products grouped by expert: argument block and row-range search
// shared by the grouped and 4-bit kernels.
#pragma once

#include "common.h"

namespace pdmb {

// Rows of group e: [ends[e-1], ends[e]) of the T activation rows (ends[-1] = 0).
// kind kRows:   C[r] = A[r] @ B[e]           A [T,K] (lda), B[e] at e * sB, C [T,N] (ldc)
// kind kReduce: C[e] = A_e^T @ B_e           A [T,M] (lda), B [T,N] (ldb), C[e] [M,N] at e * sC
// Strides in elements.
struct GroupArgs {
  const void* A;
  const void* B;
  void* C;
  const void* ends;  // E running ends, int32 or (ends64) int64
  int ends64;
  int E, T;
  int M, N, K;       // kRows: N, K; kReduce: M, N
  long long lda, ldb, ldc, sB, sC;
  int tiles_m, tiles_n;  // kReduce: tiles of one C[e]; kRows: tiles_n
  int zero_tail;     // kRows: write zeros to the rows behind the last group
};

// End of group e, held inside [0, T] so that no value of `ends` addresses
// memory outside the operands (-1 is the start of group 0).
__device__ __forceinline__ int group_end(const void* ends, int ends64, int T, int e) {
  if (e < 0) return 0;
  const long long v = ends64 ? ((const long long*)ends)[e] : (long long)((const int*)ends)[e];
  return (int)(v < 0 ? 0 : v > T ? T : v);
}

// v of the lane CTRL names, 0 where there is none (or ROWS leaves the lane out).
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int from_lane(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {  // inclusive sum over 64 lanes
  v += from_lane<0x111>(v);       // 1, 2, 4, 8 lanes back inside a row of 16
  v += from_lane<0x112>(v);
  v += from_lane<0x114>(v);
  v += from_lane<0x118>(v);
  v += from_lane<0x142, 0xa>(v);  // lane 15 of a row to the next row (rows 1, 3)
  v += from_lane<0x143, 0xc>(v);  // lane 31 to rows 2, 3
  return v;
}

// One BM-row tile of a group (e == E: the rows behind the last group).
struct RowTile {
  int e, row0, rows;  // first row, rows of it in this tile (1 .. BM)
};

// Groups [c0, c0 + 64), one a lane: first row, row count and tiles of BM rows, all
// from one load; `carry` is the end of group c0 - 1 and becomes that of c0 + 63.
struct LaneGroup {
  int lo, n, tiles;
};
template <int BM>
__device__ __forceinline__ LaneGroup lane_group(const GroupArgs& a, int c0, int lane, int& carry) {
  const int e = c0 + lane;
  int hi = group_end(a.ends, a.ends64, a.T, min(e, a.E - 1));
  hi = e < a.E ? hi : a.T;
  LaneGroup l;
  const int before = from_lane<0x138>(hi);  // (by every lane: an idle one has nothing to read)
  l.lo = lane ? before : carry;
  carry = __builtin_amdgcn_readlane(hi, 63);
  l.n = e < a.E + (a.zero_tail ? 1 : 0) ? max(hi - l.lo, 0) : 0;
  l.tiles = (l.n + BM - 1) / BM;
  return l;
}

// Number of the row tile x column tile product that block b works on, of total x
// tiles_n; false where it has none. Products are dealt to the XCDs (blocks b and b
// + 8 share one) in runs of up to 32, so that an XCD's 32 CUs work on 8 row tiles
// x 4 column tiles and its L2 serves each operand panel to several of them.
__device__ __forceinline__ bool product_of(unsigned total, unsigned tiles_n, unsigned b, int& slot, int& tn) {
  const unsigned prods = total * tiles_n;
  const unsigned per = (prods + 7) / 8, x = b & 7, i = b >> 3;
  if (i >= per) return false;
  const unsigned full = per / 32 * 32;
  const unsigned L = i < full ? (i / 32) * 256 + x * 32 + i % 32 : full * 8 + x * (per - full) + (i - full);
  if (L >= prods) return false;
  const unsigned sg = L / (8u * tiles_n), s0 = sg * 8;
  const unsigned gm = min(8u, total - s0), rem = L - sg * 8u * tiles_n;
  tn = (int)(rem / gm);
  slot = (int)(s0 + rem % gm);
  return true;
}

// The tile that `slot` of the groups in l is, `base` slots before them; inc: prefix sums of l.tiles.
template <int BM>
__device__ __forceinline__ RowTile pick_tile(const LaneGroup& l, int inc, int slot, int base, int c0) {
  const int k = __builtin_ctzll(__ballot(slot < base + inc));  // first lane whose tiles reach slot
  const int off = (slot - base - __builtin_amdgcn_readlane(inc, k) + __builtin_amdgcn_readlane(l.tiles, k)) * BM;
  return RowTile{c0 + k, __builtin_amdgcn_readlane(l.lo, k) + off, min(BM, __builtin_amdgcn_readlane(l.n, k) - off)};
}

// Block b's tile. Every wave of the workgroup searches by itself (no barrier): a
// lane takes a group, a 64-lane prefix sum gives the tiles before it; more than
// 64 groups go by 64 a pass.
template <int BM>
__device__ __forceinline__ bool find_tile(const GroupArgs& a, unsigned b, int lane, RowTile& r, int& tn) {
  int carry = 0;
  LaneGroup l = lane_group<BM>(a, 0, lane, carry);
  int inc = wave_scan(l.tiles);
  int total = __builtin_amdgcn_readlane(inc, 63);
  for (int c0 = 64; c0 < a.E + 1; c0 += 64)  // (the tail counts as a group)
    total += __builtin_amdgcn_readlane(wave_scan(lane_group<BM>(a, c0, lane, carry).tiles), 63);
  int slot;
  if (!product_of((unsigned)total, (unsigned)a.tiles_n, b, slot, tn)) return false;
  int base = 0, c0 = 0;
  for (;;) {
    const int tot = __builtin_amdgcn_readlane(inc, 63);
    if (slot < base + tot) break;
    base += tot;
    if (c0 > a.E) return false;  // (only if `ends` is written meanwhile: the search ends all the same)
    if (c0 == 0) carry = group_end(a.ends, a.ends64, a.T, min(63, a.E - 1));
    c0 += 64;
    l = lane_group<BM>(a, c0, lane, carry);
    inc = wave_scan(l.tiles);
  }
  r = pick_tile<BM>(l, inc, slot, base, c0);
  return true;
}

// Row tiles that a launch has to provide for: every group may end in a part
// of a tile, and so may the rows behind the last one.
inline long long row_tiles_bound(int T, int E, int BM, bool tail) {
  const long long g = (long long)E + (tail ? 1 : 0);
  return (long long)T / BM + (g < T ? g : T);
}

// The large-tile kernel of 16-bit products (grouped_w4.hip): whether its loads
// and offsets fit the problem, and its launch.
bool grouped_w4_ok(const GroupArgs& a, bool red, bool colmajor);
hipError_t grouped_w4(const GroupArgs& a, int dtype, bool red, bool colmajor, hipStream_t s);

}  // namespace pdmb
