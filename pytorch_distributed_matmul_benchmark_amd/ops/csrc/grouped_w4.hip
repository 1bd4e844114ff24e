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
// Both give the same register fragment, so the K-loop is one:
//   Bar0:    B(t+1) landed (vmcnt 16), every wave done reading A(t)
//   blocks 0-3 of A: 64 MFMAs | read B(t+1)'s fragments | DMA A(t+2)
//   Bar_mid: A(t+1) landed, every wave done reading B(t+1)
//   blocks 4-7: 64 MFMAs | read A(t+1)'s fragments | DMA B(t+3)
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
constexpr int LDS = 2 * REGION + 4 * kEpiBuf;

template <int DT>
__device__ __forceinline__ void mfma_acc(f32x4& acc, const s16x8& b, const s16x8& a) {
  if constexpr (DT == kBF16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}

// One LDS-DMA piece (64 lanes x 16 B) to lds0w + OFF, lane offsets only. The
// s_nop keeps 5 wait states between an SGPR restored by v_readlane and the load.
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

// One operand's panel source and fragment addresses.
template <bool KC>
struct Operand {
  u32x4 rs;             // KC: descriptor at k = 0
  const char* p;        // KS: k = 0 at the tile's first column
  long long bytes;      // KS: from p to the end of the operand
  uint32_t ld2;         // leading stride in bytes
  uint32_t voff, vlast;  // KC: lane's DMA offset, and in the last K-tile; KS: voff
  uint32_t foff[KC ? 2 : 4];  // fragment addresses in LDS: KC [ks], KS [unit & 3]

  // w2: which 128 of the 256 rows this wave's fragments are; kt: k in the last K-tile
  __device__ __forceinline__ void init(const char* base, long long ld, int rows, int ks, int wu, int lane, int w2,
                                       uint32_t region) {
    ld2 = (uint32_t)(ld * 2);
    const int l16 = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int r = wu * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
      rs = make_rsrc(base, ((long long)(min(rows, 256) - 1) * ld + ks) * 2);
      voff = r * ld2 + c * 16;
      vlast = c * 8 < ks - (ks - 1) / BK * BK ? voff : 0x80000000u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        foff[h] = region + (w2 * 128 + l16) * 128 + (((4 * h + g) ^ ((l16 >> 1) & 7)) * 16);
        asm volatile("" : "+v"(foff[h]));  // opaque: its own register
      }
    } else {
      const int k = wu * 4 + (lane >> 4), s = (k & 3) | (((k >> 3) & 1) << 2);
      const int at = (((lane & 15) >> 1) ^ s) * 16 + (lane & 1) * 8;
      p = base;
      bytes = ((long long)(ks - 1) * ld + rows) * 2;
      voff = k * ld2 + ((at / 64) * 128 + at % 64) * 2;
      const int q4 = l16 >> 2, p4 = l16 & 3, sw = q4 | ((g & 1) << 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        foff[j] = region + (8 * g + q4) * 256 + (((4 * w2 + j) ^ sw) * 32) + p4 * 8;
        asm volatile("" : "+v"(foff[j]));
      }
    }
  }
  // Descriptor of a K-tile (KS moves the base: the k axis may span more than 4 GiB).
  __device__ __forceinline__ u32x4 at(int t) const {
    if constexpr (KC) return rs;
    else {
      const long long off = (long long)t * (BK * (long long)ld2);
      return make_rsrc(p + off, bytes - off);
    }
  }
  // Lane offset of K-tile t (KC).
  __device__ __forceinline__ uint32_t base(int t, int nk) const {
    if constexpr (KC) return (t == nk - 1 ? vlast : voff) + (uint32_t)t * (BK * 2);
    else return voff;
  }
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

template <bool AKC, bool BKC>
struct Ctx {
  Operand<AKC> A;
  Operand<BKC> B;
  int nk;
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

// K-tile t from stage S; S ^ 1 holds t+1.
template <int DT, int S, bool AKC, bool BKC>
__device__ __forceinline__ void ktile(const Ctx<AKC, BKC>& c, const char* smem, int t, f32x4 (&acc)[8][8],
                                      Frag (&A)[8], Frag& A7c, Frag& A7n, Frag (&Bc)[8], Frag (&Bn)[8]) {
  constexpr int N = S ^ 1;
  const int ta = min(t + 2, c.nk - 1), tb = min(t + 3, c.nk - 1);  // clamped tail DMAs (harmless re-reads)
  const u32x4 ra = c.A.at(ta), rb = c.B.at(tb);
  const uint32_t va = c.A.base(ta, c.nk), vb = c.B.base(tb, c.nk);
#pragma unroll
  for (int mi = 0; mi < 8; ++mi) {
    if (mi == 0 || mi == 4) {
      asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int gap = 0; gap < 16; ++gap) {
      const int ks = gap >> 3, ni = gap & 7;
      mfma_acc<DT>(acc[mi][ni], Bc[ni].k[ks], mi == 7 ? A7c.k[ks] : A[mi].k[ks]);
      const int it = kItems[mi][gap];
      if (it == 1) {
        const int h = piece_of(mi, gap);  // 0..7: A of t+2 into S; 8..15: B of t+3 into S ^ 1
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

template <int DT, bool RED, bool BKC>
__global__ void __launch_bounds__(NT, 1) gemm_grouped_w4(GroupArgs a) {
  constexpr bool AKC = !RED;
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wu = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wu >> 1, wc = wu & 1;

  const char *Ap, *Bp;
  char* Cp;
  int rows, cols, ks;  // rows and columns of C left, the sum's length
  if constexpr (RED) {
    const int per = a.tiles_m * a.tiles_n;
    const int e = blockIdx.x / per, t = blockIdx.x - e * per;
    const int m0 = t / a.tiles_n * BM, n0 = t % a.tiles_n * BN;
    const int r0 = group_end(a.ends, a.ends64, a.T, e - 1), r1 = group_end(a.ends, a.ends64, a.T, e);
    ks = __builtin_amdgcn_readfirstlane(r1 > r0 ? r1 - r0 : 0);
    rows = a.M - m0;
    cols = a.N - n0;
    const long long r0u = __builtin_amdgcn_readfirstlane(r0);
    Ap = (const char*)a.A + (r0u * a.lda + m0) * 2;
    Bp = (const char*)a.B + (r0u * a.ldb + n0) * 2;
    Cp = (char*)a.C + ((long long)e * a.sC + (long long)m0 * a.ldc + n0) * 2;
  } else {
    RowTile r;
    int tn;
    if (!find_tile<BM>(a, blockIdx.x, lane, r, tn)) return;
    const bool zero = r.e == a.E;
    ks = zero ? 0 : a.K;
    rows = r.rows;
    cols = a.N - tn * BN;
    Ap = (const char*)a.A + (long long)r.row0 * a.lda * 2;
    Bp = (const char*)a.B + ((long long)(zero ? 0 : r.e) * a.sB + (long long)tn * BN * (BKC ? a.ldb : 1)) * 2;
    Cp = (char*)a.C + ((long long)r.row0 * a.ldc + (long long)tn * BN) * 2;
  }

  const long long ldc2 = a.ldc * 2;
  if (ks <= 0) {  // an empty sum (8-byte zeros: columns come in groups of 4 or more)
    const int nr = min(rows, BM), nc = min(cols, BN) / 4;
    for (int r = wu; r < nr; r += 4)
      if (lane < nc) *(u32x2*)(Cp + r * ldc2 + lane * 8) = u32x2{0u, 0u};
    return;
  }
  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  {
    Ctx<AKC, BKC> c;
    c.nk = (ks + BK - 1) / BK;
    c.lds0w = (uint32_t)(size_t)((lds_void*)smem) + wu * 1024;
    c.A.init(Ap, a.lda, rows, ks, wu, lane, wr, 0);
    c.B.init(Bp, a.ldb, cols, ks, wu, lane, wc, REGION);

    // The DMA order that the loop's counted waits assume: A(0), B(0) to stage 0, B(1),
    // A(1) to stage 1; tile 0's fragments to registers; B(2) to stage 0.
    const int nk = c.nk, t1 = min(1, nk - 1), t2 = min(2, nk - 1);
    {
      const u32x4 ra0 = c.A.at(0), rb0 = c.B.at(0), ra1 = c.A.at(t1), rb1 = c.B.at(t1);
      const uint32_t va0 = c.A.base(0, nk), vb0 = c.B.base(0, nk), va1 = c.A.base(t1, nk), vb1 = c.B.base(t1, nk);
#pragma unroll
      for (int h = 0; h < 8; ++h) c.A.piece(ra0, va0, c.lds0w, 0, h);
#pragma unroll
      for (int h = 0; h < 8; ++h) c.B.piece(rb0, vb0, c.lds0w, REGION, h);
#pragma unroll
      for (int h = 0; h < 8; ++h) c.B.piece(rb1, vb1, c.lds0w, REGION + PANEL, h);
#pragma unroll
      for (int h = 0; h < 8; ++h) c.A.piece(ra1, va1, c.lds0w, PANEL, h);
    }
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");  // tile 0 landed everywhere
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
      const u32x4 rb2 = c.B.at(t2);
      const uint32_t vb2 = c.B.base(t2, nk);
#pragma unroll
      for (int h = 0; h < 8; ++h) c.B.piece(rb2, vb2, c.lds0w, REGION, h);
    }
    int t = 0;
    for (; t + 1 < nk; t += 2) {  // branch-free body: the fragment sets swap roles every K-tile
      ktile<DT, 0>(c, smem, t, acc, A, A7a, A7b, B0, B1);
      ktile<DT, 1>(c, smem, t + 1, acc, A, A7b, A7a, B1, B0);
    }
    if (t < nk) ktile<DT, 0>(c, smem, t, acc, A, A7a, A7b, B0, B1);
    // Tail DMAs landed; the last MFMAs (asm: unseen by the hazard recognizer) have written.
    asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
  }

  // C leaves through LDS as whole rows (common.h store_block16), past the stages.
  char* ebuf = smem + 2 * REGION + wu * kEpiBuf;
  const bool inside = rows >= BM && cols >= BN;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f32x4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = acc[i][j];
    if (inside) store_block16<DT, false, false>(ebuf, v, 1.0f, Cp, ldc2, wr * 128 + i * 16, wc * 128, rows, cols, lane);
    else store_block16<DT, true, false>(ebuf, v, 1.0f, Cp, ldc2, wr * 128 + i * 16, wc * 128, rows, cols, lane);
  }
}

template <int DT, bool RED, bool BKC>
hipError_t launch(GroupArgs a, hipStream_t s) {
  a.tiles_m = (a.M + BM - 1) / BM;
  a.tiles_n = (a.N + BN - 1) / BN;
  const long long blocks =
      RED ? (long long)a.E * a.tiles_m * a.tiles_n
          : (row_tiles_bound(a.T, a.E, BM, a.zero_tail) * a.tiles_n + 7) / 8 * 8;
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_grouped_w4<DT, RED, BKC>), dim3((unsigned)blocks), dim3(NT), 0, s, a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(const GroupArgs& a, bool red, bool colmajor, hipStream_t s) {
  return red ? launch<DT, true, false>(a, s) : colmajor ? launch<DT, false, true>(a, s) : launch<DT, false, false>(a, s);
}

}  // namespace kgw4

bool grouped_w4_ok(const GroupArgs& a, bool red, bool colmajor) {
  auto al = [](const void* p, long long ld, long long batch) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && batch % 8 == 0;
  };
  // lane offsets stay below 2^31: 256 rows (KC) or 64 (KS) of one panel, and a row's length
  const long long span = 1ll << 21;
  return al(a.A, a.lda, 0) && al(a.B, a.ldb, a.sB) && (uintptr_t)a.C % 8 == 0 && a.ldc % 4 == 0 && a.sC % 4 == 0 &&
         a.lda <= span && a.ldb <= span && a.N % 8 == 0 && (red ? a.M % 8 == 0 : a.K % 8 == 0);
}

hipError_t grouped_w4(const GroupArgs& a, int dtype, bool red, bool colmajor, hipStream_t s) {
  return dtype == kBF16 ? kgw4::launch_dt<kBF16>(a, red, colmajor, s) : kgw4::launch_dt<kF16>(a, red, colmajor, s);
}

}  // namespace pdmb
