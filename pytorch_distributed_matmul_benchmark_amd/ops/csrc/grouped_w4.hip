// grouped_w4.hip — the grouped products' large-tile kernel, bf16 / fp16: 256 x
// 256 x 64 tiles, 4 waves per workgroup, one per SIMD, each owning 128 x 128
// outputs in 256 AGPR accumulators, operands staged by LDS-DMA two K-tiles
// ahead. One template serves both products (grouped.hip):
//   rows:   A = the rows (KC), B = the expert's weight, row-major (KS) or column-major (KC)
//   reduce: A and B are the two row matrices, both KS, the K axis is the group's rows
// KC = k contiguous, KS = k strided; an operand panel of a K-tile is 32 KiB:
//   KC  [256 rows][128 B], 16-B chunk c of a row at c ^ ((row >> 1) & 7); ds_read_b128.
//   KS  two halves [64 k][256 B] of 128 columns (half q: columns 128 i + 64 q .. + 63),
//       32-B unit u at u ^ ((k & 3) | ((k >> 3) & 1) << 2); ds_read_b64_tr_b16.
// Both give the same register fragment, so the K-loop is one. K-tile s of the
// stream, from LDS stage s & 1 (its fragments are in registers already):
//   Bar0:    B(s+1) landed, every wave done reading A(s)
//   blocks 0-3 of A: 64 MFMAs | read B(s+1)'s fragments | DMA A(s+2)
//   Bar_mid: A(s+1) landed, every wave done reading B(s+1)
//   blocks 4-7: 64 MFMAs | read A(s+1)'s fragments | DMA B(s+3)
//
// A stream: a workgroup, one a CU, runs its tiles (b, b + grid, ...) as one
// sequence of K-tiles. What the loop fetches two and three K-tiles ahead is the
// next tile's where this one ends, so a tile's first loads and the last one's
// stores cost no time of their own (16384 rows of 8 experts, 4096 x 8192: 890 us one
// tile a workgroup, 851 streamed, 1290 TFLOP/s: matrix units and their power; a training
// step of 8192 rows of 8, 4096 x 4096: 802, 765, where three products of 9 rounds' tiles over
// 4 waste an eighth and the weight gradients' stores come in bursts). A tile has an even
// number of K-tiles, four at least (beyond its
// sum's end they are zeros): stages and fragment sets then have the same roles at
// every tile's start, which hipcc's register allocation needs, and only the next tile is ever
// looked at.
//
// The stores: 32 a wave and tile, always — those of rows or columns that C has not
// go past the buffer's end —, and vmcnt counts loads and stores in order, so a tile's first
// three waits leave 16 + 32 operations in flight where the others leave 16 (the first
// tile has 32 stores that go nowhere before it).
//
// Edges without masks in the loop: every DMA offset is in the lane's offset
// register (a scalar offset is not part of the descriptor's range check), so
// rows past a group's last one, k past the end of a KS panel, and columns
// past the matrix' end read as zeros; k past the end of a KC row is steered out of the
// descriptor by a second offset register that the last K-tile uses. A partial
// last K-tile is therefore zeros in both operands, whatever lies beside them in memory.
//
// The two panels of an operand are 32 KiB apart, so one register a fragment
// address serves both stages (the rest is in the instructions' 16-bit offsets).
#include "api.h"
#include "grouped.h"

namespace pdmb {
namespace kgw4 {

constexpr int BM = 256, BN = 256, BK = 64, NT = 256;
constexpr int PANEL = 256 * BK * 2;   // 32 KiB
constexpr int REGION = 2 * PANEL;     // an operand's two stages
constexpr int kMaxGroups = 14 * 64;   // 1 KiB of LDS for 64 groups
constexpr int LDS = 2 * REGION + 4 * kEpiBuf + kMaxGroups / 64 * 1024;
static_assert(LDS <= 160 * 1024, "LDS");

template <int DT>
__device__ __forceinline__ void mfma_acc(f32x4& acc, const s16x8& b, const s16x8& a) {
  if constexpr (DT == kBF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}

// The first MFMA of a tile: C = 0. (In place, so that the accumulators keep their registers.)
template <int DT>
__device__ __forceinline__ void mfma_first(f32x4& acc, const s16x8& b, const s16x8& a) {
  if constexpr (DT == kBF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "+a"(acc) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "+a"(acc) : "v"(b), "v"(a));
}

// One LDS-DMA piece (64 lanes x 16 B) to lds0w + OFF, lane offsets only. The
// s_nop keeps 5 wait states between an SGPR restored by v_readlane and the load: the next tile's
// operands and the search do not fit beside the loop's descriptors where an operand is KS, and 20 (row-major B)
// or 47 (reduce) SGPRs wait in lanes of a vector register. No vector register spills.
__device__ __forceinline__ void dma_piece(u32x4 rsrc, uint32_t voff, uint32_t lds0w, int off) {
  asm volatile(
      "s_add_u32 m0, %2, %3\n\t"
      "s_nop 3\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(rsrc), "s"(lds0w), "i"(off)
      : "memory", "m0", "scc");
}

struct Frag {  // one 16-row block of a K-tile: k 0..31 and 32..63
  s16x8 k[2];
};

// One operand of a tile: where its k = 0 is.
template <bool KC>
struct Source {
  u32x4 rs;         // KC: descriptor of the tile's rows
  const char* p;    // KS: first column, k = 0
  long long bytes;  // KS: from p to the end of the operand
  __device__ __forceinline__ void set(const char* base, long long ld, int rows, int ks) {
    if constexpr (KC) {
      rs = make_rsrc(base, ((long long)(min(rows, 256) - 1) * ld + ks) * 2);
    } else {
      p = base;
      bytes = ks > 0 ? ((long long)(ks - 1) * ld + rows) * 2 : 0;
    }
  }
};

// What a lane knows of an operand, whatever the tile.
template <bool KC>
struct Operand {
  uint32_t ld2;               // leading stride in bytes
  int last;                   // KC: the last K-tile with any k
  uint32_t voff, vlast;       // DMA offset of piece 0; KC: and in that K-tile
  uint32_t foff[KC ? 2 : 4];  // fragment addresses in LDS: KC [ks], KS [unit & 3]

  // w2: which 128 of the 256 rows this wave's fragments are; KC: ks is every tile's
  __device__ __forceinline__ void init(long long ld, int ks, int wu, int lane, int w2, uint32_t region) {
    ld2 = (uint32_t)(ld * 2);
    last = (ks - 1) / BK;
    const int l16 = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int r = wu * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
      voff = r * ld2 + c * 16;
      vlast = c * 8 < ks - last * BK ? voff : 0x80000000u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        foff[h] = region + (w2 * 128 + l16) * 128 + (((4 * h + g) ^ ((l16 >> 1) & 7)) * 16);
        asm volatile("" : "+v"(foff[h]));  // opaque: its own register
      }
    } else {
      const int k = wu * 4 + (lane >> 4), s = (k & 3) | (((k >> 3) & 1) << 2);
      const int at = (((lane & 15) >> 1) ^ s) * 16 + (lane & 1) * 8;
      voff = k * ld2 + ((at / 64) * 128 + at % 64) * 2;
      vlast = voff;
      const int q4 = l16 >> 2, p4 = l16 & 3, sw = q4 | ((g & 1) << 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        foff[j] = region + (8 * g + q4) * 256 + (((4 * w2 + j) ^ sw) * 32) + p4 * 8;
        asm volatile("" : "+v"(foff[j]));
      }
    }
  }
  // Descriptor of K-tile t (KS moves the base: the k axis may span more than 4 GiB).
  __device__ __forceinline__ u32x4 at(const Source<KC>& s, int t) const {
    if constexpr (KC) return s.rs;
    else {
      const long long off = (long long)t * (BK * (long long)ld2);
      return make_rsrc(s.p + off, s.bytes - off);
    }
  }
  // K-tile t of this tile, or the next one's (here false): scalar selects, no branch.
  __device__ __forceinline__ u32x4 at(const Source<KC>& cur, const Source<KC>& nxt, bool here, int t) const {
    Source<KC> s;
    if constexpr (KC) {
      s.rs.x = here ? cur.rs.x : nxt.rs.x;
      s.rs.y = here ? cur.rs.y : nxt.rs.y;
      s.rs.z = here ? cur.rs.z : nxt.rs.z;
      s.rs.w = cur.rs.w;
    } else {
      s.p = here ? cur.p : nxt.p;
      s.bytes = here ? cur.bytes : nxt.bytes;
    }
    return at(s, t);
  }
  // Lane offset of K-tile t, and of one before the sum's last two (KC: k past the end reads as zeros).
  __device__ __forceinline__ uint32_t base(int t) const {
    if constexpr (KC) return (t < last ? voff : t == last ? vlast : 0x80000000u) + (uint32_t)t * (BK * 2);
    else return voff;
  }
  __device__ __forceinline__ uint32_t inner(int t) const { return KC ? voff + (uint32_t)t * (BK * 2) : voff; }
  // DMA piece h (0..7): KC rows 32 h + 8 wu .. + 7, KS half h >> 2, k 16 (h & 3) + 4 wu .. + 3.
  __device__ __forceinline__ void piece(u32x4 r, uint32_t v, uint32_t lds0w, int panel, int h) const {
    if constexpr (KC) dma_piece(r, v + (uint32_t)(h * 32) * ld2, lds0w, panel + h * 4096);
    else dma_piece(r, v + (uint32_t)((h & 3) * 16) * ld2 + (h >> 2) * 128, lds0w,
                   panel + (h >> 2) * 16384 + (h & 3) * 4096);
  }
  // Half ks of the fragment of 16-row block m from stage st.
  __device__ __forceinline__ s16x8 frag(const char* smem, int st, int m, int ks) const {
    if constexpr (KC) {
      return *(const lds_s16x8*)(smem + foff[ks] + st * PANEL + m * 2048);
    } else {
      const char* q = smem + foff[m & 3] + st * PANEL + (m >> 2) * 16384 + ks * 8192;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 1024));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// An output tile: operands, length of the sum in K-tiles (even, 4 at least), and C's part of it.
template <bool AKC, bool BKC>
struct OutTile {
  Source<AKC> A;
  Source<BKC> B;
  char* C;
  int rows, cols, nk;
};

template <bool AKC, bool BKC>
struct Ctx {
  Operand<AKC> A;
  Operand<BKC> B;
  uint32_t lds0w;  // LDS address of the wave's 1 KiB of a piece
};

// What follows MFMA `gap` (ks * 8 + ni) of A block `blk`. 1: the next DMA piece;
// 100 + 2 s + ks: B fragment half of tile t+1; 200 + 2 m + ks: A fragment
// half of t+1 (m = 7: into the second A7 set). A block m of t+1 is read only after
// block m of t is used up.
constexpr int kItems[8][16] = {
    {100, 0, 101, 0, 1, 0, 102, 0, 103, 0, 1, 0, 0, 0, 0, 0},
    {104, 0, 105, 0, 1, 0, 106, 0, 107, 0, 1, 0, 0, 0, 0, 0},
    {108, 0, 109, 0, 1, 0, 110, 0, 111, 0, 1, 0, 0, 0, 0, 0},
    {112, 0, 113, 0, 1, 0, 114, 0, 115, 0, 1, 0, 0, 0, 0, 0},
    {200, 0, 201, 0, 1, 0, 202, 0, 203, 0, 1, 0, 0, 0, 0, 0},
    {204, 0, 205, 0, 1, 0, 206, 0, 207, 0, 1, 0, 0, 0, 0, 0},
    {208, 0, 209, 0, 1, 0, 210, 0, 211, 0, 1, 0, 214, 0, 215, 0},
    {212, 0, 213, 0, 1, 0, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0}};

constexpr int piece_of(int blk, int gap) {  // running index of a DMA item (0..15)
  int n = 0;
  for (int b = 0; b < 8; ++b)
    for (int g = 0; g < 16; ++g) {
      if (b == blk && g == gap) return n;
      if (kItems[b][g] == 1) ++n;
    }
  return n;
}

// K-tile t of `cur` from stage S; stage S ^ 1 holds the stream's next one. W0, W1: operations
// in flight at its barriers; ZERO: starts the sums; SEL: what it fetches may be the next tile's.
template <int DT, int S, int W0, int W1, bool ZERO, bool SEL, bool AKC, bool BKC>
__device__ __forceinline__ void ktile(const Ctx<AKC, BKC>& c, const OutTile<AKC, BKC>& cur,
                                      const OutTile<AKC, BKC>& nxt, bool more, const char* smem, int t,
                                      f32x4 (&acc)[8][8], Frag (&A)[8], Frag& A7c, Frag& A7n, Frag (&Bc)[8],
                                      Frag (&Bn)[8]) {
  constexpr int N = S ^ 1;
  u32x4 ra, rb;
  uint32_t va, vb;
  if constexpr (SEL) {
    // this tile's, the next one's, or (last tile) a harmless re-read
    const bool ha = t + 2 < cur.nk || !more, hb = t + 3 < cur.nk || !more;
    const int ta = ha ? min(t + 2, cur.nk - 1) : t + 2 - cur.nk, tb = hb ? min(t + 3, cur.nk - 1) : t + 3 - cur.nk;
    ra = c.A.at(cur.A, nxt.A, ha, ta);
    rb = c.B.at(cur.B, nxt.B, hb, tb);
    va = c.A.base(ta);
    vb = c.B.base(tb);
  } else {
    ra = c.A.at(cur.A, t + 2);
    rb = c.B.at(cur.B, t + 3);
    va = c.A.inner(t + 2);
    vb = c.B.inner(t + 3);
  }
#pragma unroll
  for (int mi = 0; mi < 8; ++mi) {
    if (mi == 0 || mi == 4) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(mi == 0 ? W0 : W1) : "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int gap = 0; gap < 16; ++gap) {
      const int ks = gap >> 3, ni = gap & 7;
      if (ZERO && ks == 0) mfma_first<DT>(acc[mi][ni], Bc[ni].k[ks], mi == 7 ? A7c.k[ks] : A[mi].k[ks]);
      else mfma_acc<DT>(acc[mi][ni], Bc[ni].k[ks], mi == 7 ? A7c.k[ks] : A[mi].k[ks]);
      const int it = kItems[mi][gap];
      if (it == 1) {
        const int h = piece_of(mi, gap);  // 0..7: A of s+2 into S; 8..15: B of s+3 into S ^ 1
        if (h < 8) c.A.piece(ra, va, c.lds0w, S * PANEL, h);
        else c.B.piece(rb, vb, c.lds0w, REGION + N * PANEL, h - 8);
      } else if (it >= 100 && it < 200) {
        const int s = (it - 100) >> 1, h = (it - 100) & 1;
        Bn[s].k[h] = c.B.frag(smem, N, s, h);
      } else if (it >= 214) {
        A7n.k[it - 214] = c.A.frag(smem, N, 7, it - 214);
      } else if (it >= 200) {
        const int m = (it - 200) >> 1, h = (it - 200) & 1;
        A[m].k[h] = c.A.frag(smem, N, m, h);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// C leaves through this wave's LDS buffer as whole rows: 32 stores of 4 rows x 256 B.
template <int DT, bool AKC, bool BKC>
__device__ __forceinline__ void store_tile(const OutTile<AKC, BKC>& o, f32x4 (&acc)[8][8], char* ebuf, int ldc2,
                                           int wr, int wc, int tid) {
  typedef __attribute__((address_space(3))) char lds_char;
  constexpr int P = epi_pitch<8>();
  int lane = tid & 63;
  asm volatile("" : "+v"(lane));  // formed here: nothing of it lives through the K-loop
  const int l16 = lane & 15, g = lane >> 4;
  lds_char* lb = (lds_char*)(lds_void*)ebuf;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(o.C, 0, 0x7fffffff, 0x00020000);
  const int col = wc * 128 + 8 * l16, left = o.rows - wr * 128 - g;  // rows of C from this lane's first one
  const int voff = col < o.cols ? (wr * 128 + g) * ldc2 + col * 2 : (int)0x80000000;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+a"(acc[i][j]));  // read here, not sooner
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *(lds_u32x2*)(lb + l16 * P + (j * 16 + 4 * g) * 2) =
          u32x2{pack2<DT>(acc[i][j].x, acc[i][j].y), pack2<DT>(acc[i][j].z, acc[i][j].w)};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const u32x4 x = *(lds_u32x4_t*)(lb + (g + 4 * r) * P + l16 * 16);
      const int v = 16 * i + 4 * r < left ? voff : (int)0x80000000;
      __builtin_amdgcn_raw_buffer_store_b128(x, rs, v, (16 * i + 4 * r) * ldc2, 2 /* nt */);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int DT, bool RED, bool BKC>
__global__ void __launch_bounds__(NT, 1) gemm_grouped_w4(GroupArgs a) {
  constexpr bool AKC = !RED;
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wu = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wu >> 1, wc = wu & 1;

  // Rows behind the last group: zeros, 8 bytes a lane, dealt to the workgroups.
  if (!RED && a.zero_tail) {
    const int r0 = __builtin_amdgcn_readfirstlane(group_end(a.ends, a.ends64, a.T, a.E - 1));
    for (int r = r0 + blockIdx.x; r < a.T; r += gridDim.x)
      for (int n = tid * 4; n < a.N; n += NT * 4)
        *(u32x2*)((char*)a.C + ((long long)r * a.ldc + n) * 2) = u32x2{0u, 0u};
  }

  // The groups' tiles stay in LDS for the whole stream: first rows, row counts, tile counts
  // and their prefix sums of 64 groups a KiB.
  typedef __attribute__((address_space(3))) int lds_int;
  lds_int* kept = (lds_int*)(lds_void*)(smem + 2 * REGION + 4 * kEpiBuf);
  for (int c = wu; c * 64 < a.E; c += 4) {
    int carry = __builtin_amdgcn_readfirstlane(group_end(a.ends, a.ends64, a.T, c * 64 - 1));
    GroupArgs g = a;
    g.zero_tail = 0;
    const LaneGroup l = lane_group<BM>(g, c * 64, lane, carry);
    kept[c * 256 + lane] = l.lo;
    kept[c * 256 + 64 + lane] = l.n;
    kept[c * 256 + 128 + lane] = l.tiles;
    kept[c * 256 + 192 + lane] = wave_scan(l.tiles);
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  int total = 0;  // row tiles
  if constexpr (!RED) {
    for (int c = 0; c * 64 < a.E; ++c) total += kept[c * 256 + 255];
    total = __builtin_amdgcn_readfirstlane(total);
  }
  // Tile b of the launch's order.
  auto tile_at = [&](int b, OutTile<AKC, BKC>& o) -> bool {
    if constexpr (RED) {
      const int per = a.tiles_m * a.tiles_n;
      if (b >= a.E * per) return false;
      const int e = b / per, t = b - e * per;
      const int m0 = t / a.tiles_n * BM, n0 = t % a.tiles_n * BN;
      const int at = (e >> 6) * 256 + (e & 63);
      const int r0 = __builtin_amdgcn_readfirstlane(kept[at]), ks = __builtin_amdgcn_readfirstlane(kept[at + 64]);
      o.rows = a.M - m0;
      o.cols = a.N - n0;
      o.nk = max((ks + 2 * BK - 1) / (2 * BK) * 2, 4);
      o.A.set((const char*)a.A + ((long long)r0 * a.lda + m0) * 2, a.lda, o.rows, ks);
      o.B.set((const char*)a.B + ((long long)r0 * a.ldb + n0) * 2, a.ldb, o.cols, ks);
      o.C = (char*)a.C + ((long long)e * a.sC + (long long)m0 * a.ldc + n0) * 2;
    } else {
      int tn, slot, base = 0, c = 0;
      if (!product_of((unsigned)total, (unsigned)a.tiles_n, (unsigned)b, slot, tn)) return false;
      int ln = tid & 63;
      asm volatile("" : "+v"(ln));  // formed here: nothing of it lives through the K-loop
      for (;; ++c) {
        const int tot = __builtin_amdgcn_readfirstlane(kept[c * 256 + 255]);
        if (slot < base + tot) break;
        base += tot;
      }
      const lds_int* k = kept + c * 256 + ln;
      const RowTile r = pick_tile<BM>(LaneGroup{k[0], k[64], k[128]}, k[192], slot, base, c * 64);
      o.rows = r.rows;
      o.cols = a.N - tn * BN;
      o.nk = (a.K + 2 * BK - 1) / (2 * BK) * 2;
      o.A.set((const char*)a.A + (long long)r.row0 * a.lda * 2, a.lda, o.rows, a.K);
      o.B.set((const char*)a.B + ((long long)r.e * a.sB + (long long)tn * BN * (BKC ? a.ldb : 1)) * 2, a.ldb, o.cols,
              a.K);
      o.C = (char*)a.C + ((long long)r.row0 * a.ldc + (long long)tn * BN) * 2;
    }
    return true;
  };

  int b = blockIdx.x;
  OutTile<AKC, BKC> cur, nxt;
  if (!tile_at(b, cur)) return;
  Ctx<AKC, BKC> c;
  c.lds0w = (uint32_t)(size_t)((lds_void*)smem) + wu * 1024;
  c.A.init(a.lda, a.K, wu, lane, wr, 0);
  c.B.init(a.ldb, a.K, wu, lane, wc, REGION);
  const int ldc2 = (int)(a.ldc * 2);
  char* ebuf = smem + 2 * REGION + wu * kEpiBuf;

  // The DMA order that the loop's counted waits assume: A(0), B(0) to stage 0, B(1),
  // A(1) to stage 1; tile 0's fragments to registers; B(2) to stage 0; 32 stores.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  {
    const u32x4 ra0 = c.A.at(cur.A, 0), rb0 = c.B.at(cur.B, 0), ra1 = c.A.at(cur.A, 1), rb1 = c.B.at(cur.B, 1);
    const uint32_t va0 = c.A.base(0), vb0 = c.B.base(0), va1 = c.A.base(1), vb1 = c.B.base(1);
#pragma unroll
    for (int h = 0; h < 8; ++h) c.A.piece(ra0, va0, c.lds0w, 0, h);
#pragma unroll
    for (int h = 0; h < 8; ++h) c.B.piece(rb0, vb0, c.lds0w, REGION, h);
#pragma unroll
    for (int h = 0; h < 8; ++h) c.B.piece(rb1, vb1, c.lds0w, REGION + PANEL, h);
#pragma unroll
    for (int h = 0; h < 8; ++h) c.A.piece(ra1, va1, c.lds0w, PANEL, h);
  }
  asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");  // K-tile 0 landed everywhere
  f32x4 acc[8][8];
  Frag A[8], A7a, A7b, B0[8], B1[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      A[i].k[h] = c.A.frag(smem, 0, i, h);
      B0[i].k[h] = c.B.frag(smem, 0, i, h);
    }
  A7a = A[7];
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // stage 0's B read by all
  {
    const u32x4 rb2 = c.B.at(cur.B, 2);
    const uint32_t vb2 = c.B.base(2);
#pragma unroll
    for (int h = 0; h < 8; ++h) c.B.piece(rb2, vb2, c.lds0w, REGION, h);
  }
  {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((char*)a.C, 0, 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{0u, 0u, 0u, 0u}, rs, (int)0x80000000, 0, 2);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (;;) {
    b += gridDim.x;
    const bool more = tile_at(b, nxt);
    // (32 stores of the tile before are in flight)
    ktile<DT, 0, 48, 48, true, true>(c, cur, nxt, more, smem, 0, acc, A, A7a, A7b, B0, B1);
    ktile<DT, 1, 48, 16, false, true>(c, cur, nxt, more, smem, 1, acc, A, A7b, A7a, B1, B0);
    int t = 2;
    // (fetches up to B's K-tile t + 4: it has to lie before the sum's last two)
    for (; t + 8 <= cur.nk; t += 2) {
      ktile<DT, 0, 16, 16, false, false>(c, cur, nxt, more, smem, t, acc, A, A7a, A7b, B0, B1);
      ktile<DT, 1, 16, 16, false, false>(c, cur, nxt, more, smem, t + 1, acc, A, A7b, A7a, B1, B0);
    }
    for (; t < cur.nk; t += 2) {
      ktile<DT, 0, 16, 16, false, true>(c, cur, nxt, more, smem, t, acc, A, A7a, A7b, B0, B1);
      ktile<DT, 1, 16, 16, false, true>(c, cur, nxt, more, smem, t + 1, acc, A, A7b, A7a, B1, B0);
    }
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");  // the asm MFMAs have written
    store_tile<DT>(cur, acc, ebuf, ldc2, wr, wc, tid);
    if (!more) break;
    cur = nxt;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // tail DMAs landed before the LDS is released
}

template <int DT, bool RED, bool BKC>
hipError_t launch(GroupArgs a, int cus, hipStream_t s) {
  a.tiles_m = (a.M + BM - 1) / BM;
  a.tiles_n = (a.N + BN - 1) / BN;
  const long long tiles = RED ? (long long)a.E * a.tiles_m * a.tiles_n
                              : (row_tiles_bound(a.T, a.E, BM, false) * a.tiles_n + 7) / 8 * 8;
  if (tiles > (1ll << 30)) return hipErrorInvalidValue;
  // a multiple of 8, so that a workgroup's tiles stay on one XCD's part of the order
  const long long grid = tiles < cus ? (tiles + 7) / 8 * 8 : cus / 8 * 8;
  hipLaunchKernelGGL((gemm_grouped_w4<DT, RED, BKC>), dim3((unsigned)grid), dim3(NT), 0, s, a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(const GroupArgs& a, bool red, bool colmajor, int cus, hipStream_t s) {
  return red        ? launch<DT, true, false>(a, cus, s)
         : colmajor ? launch<DT, false, true>(a, cus, s)
                    : launch<DT, false, false>(a, cus, s);
}

}  // namespace kgw4

bool grouped_w4_ok(const GroupArgs& a, bool red, bool colmajor) {
  auto al = [](const void* p, long long ld, long long batch) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && batch % 8 == 0;
  };
  // lane offsets stay below 2^31: 256 rows (KC) or 64 (KS) of one panel, and a row's length
  const long long span = 1ll << 21;
  return al(a.A, a.lda, 0) && al(a.B, a.ldb, a.sB) && (uintptr_t)a.C % 8 == 0 && a.ldc % 4 == 0 && a.sC % 4 == 0 &&
         a.lda <= span && a.ldb <= span && a.ldc <= span && a.N % 8 == 0 &&
         a.E <= kgw4::kMaxGroups &&
         (red ? a.M % 8 == 0 : a.K % 8 == 0 && a.K > 2 * kgw4::BK);
}

hipError_t grouped_w4(const GroupArgs& a, int dtype, bool red, bool colmajor, hipStream_t s) {
  int dev = 0, cus = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return e;
  if (cus < 8) cus = 8;
  return dtype == kBF16 ? kgw4::launch_dt<kBF16>(a, red, colmajor, cus, s)
                        : kgw4::launch_dt<kF16>(a, red, colmajor, cus, s);
}

}  // namespace pdmb
