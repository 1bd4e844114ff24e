// grouped.hip — matrix products grouped by expert with ragged sizes, bf16 /
// fp16 (fp32 accumulate) and exact fp32:
//   rows:   C[r] = A[r] @ B[e]        for the rows r of group e
//   reduce: C[e] = A_e^T @ B_e        summed over the rows of group e
// (`rows` serves the forward product and, with B transposed by its strides, the
// gradient of the rows; `reduce` is the gradient of the weights.)
//
// Operands are tiled by the two layouts an operand of an MFMA can have in
// memory: KC, k contiguous (rows of A; a column-major B), and KS, k strided (a
// row-major B; both operands of `reduce`, whose k runs over rows). A K-tile is
// 128 bytes of k (64 16-bit or 32 fp32 values). LDS images:
//   KC  [row][128 B], 16-B chunk c of a row at c ^ ((row >> 1) & 7), read by
//       ds_read_b128: lane (l16, g) takes chunk 4 h + g of row l16.
//   KS  16-bit: [k][128 columns], 32-B unit u at u ^ ((k & 3) | ((k >> 3) & 1) << 2),
//       read transposed by ds_read_b64_tr_b16. fp32: 64-B unit u at
//       u ^ ((k >> 2) & 3), read by ds_read_b32, one k a lane.
// In fp32 MFMA step (h, j) multiplies k = 16 h + 4 g + j: any order of k that
// both operands share gives the same sum of products.
//
// This kernel stages global -> registers -> LDS: PF K-tiles in flight in
// registers, two LDS stages, one barrier a K-tile. BUF: operands at a multiple
// of 4 bytes come as 16-byte buffer loads whose descriptor ends with the tile's last
// row (KC) or k (KS), moved along k, so that what is not there reads as zero with no
// branch (a branch around a load makes hipcc wait for later loads too); only a row
// that ends inside 16 bytes is masked, in its last K-tile. 16-bit operands of odd
// strides are read as the five aligned dwords around a chunk and shifted on their way
// to LDS. Strides past 8 MB are read by the element at the edges.
//
// What bounds it: with few rows the read of the weights (48 rows of 64 experts 4096 x
// 2048 bf16, 88 to 109 us by where the weights lie in memory: 5.2 to 6.4 TB/s); in 16 bits and
// with more rows the LDS pipe and the barrier a K-tile (256 x 256 tiles take over:
// grouped_w4.hip); in fp32 the matrix units, with the padding of groups to tiles (1357
// rows of 16 experts 1001 x 1416, 52 us: 74 of 152 TFLOP/s, 87 with the padding).
#include "api.h"
#include "grouped.h"

#include <cmath>

namespace pdmb {
namespace kgrp {

constexpr int NT = 256;
enum Loads { kAny, kDwords, kOdd };  // how the operands are read (above)

template <int DT>
constexpr int esize() { return DT == kF32 ? 4 : 2; }

// 16 bytes at p (any alignment), of which `avail` elements are inside the operand.
template <int DT>
__device__ __forceinline__ u32x4 load_chunk(const char* p, int avail) {
  constexpr int ES = esize<DT>(), EPC = 16 / ES;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (avail >= EPC) {
    __builtin_memcpy(&v, p, 16);
  } else if (avail > 0) {
    if constexpr (ES == 4) {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < avail) v[i] = *(const unsigned*)(p + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < avail) v[i >> 1] |= (unsigned)*(const unsigned short*)(p + 2 * i) << (16 * (i & 1));
    }
  }
  return v;
}

// The first `avail` elements of a chunk, zeros for the rest.
template <int DT>
__device__ __forceinline__ u32x4 keep(u32x4 v, int avail) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == kF32) v[i] = i < avail ? v[i] : 0u;
    else v[i] = 2 * i + 1 < avail ? v[i] : 2 * i < avail ? v[i] & 0xffffu : 0u;
  }
  return v;
}

// One operand tile of R rows (or columns) x one K-tile.
template <int DT, bool KC, int R, int BUF>
struct Tile {
  static constexpr int ES = esize<DT>(), EPC = 16 / ES, BK = 128 / ES;
  static constexpr int BYTES = R * 128;
  static constexpr int CH = (R * 8 + NT - 1) / NT;  // chunks a thread
  static constexpr int PITCH = R * ES;              // KS image: bytes of one k
  static constexpr int CPK = PITCH / 16;
  static_assert(KC || R * ES >= 256, "the KS swizzles' units");

  const char* p;   // first row / column, k = 0
  long long ld;    // leading stride
  int rows, ks;    // what there is of it
  int first;       // lane's offset of chunk 0 in bytes (BUF)
  int odd;         // kOdd: bytes of p past a dword

  __device__ __forceinline__ Tile(const char* p_, long long ld_, int rows_, int ks_, int tid)
      : p(p_), ld(ld_), rows(rows_ < R ? rows_ : R), ks(ks_), odd(BUF == kOdd ? (int)((uintptr_t)p_ & 2) : 0) {
    first = KC ? (tid >> 3) * (int)(ld * ES) + (tid & 7) * 16 : tid / CPK * (int)(ld * ES) + tid % CPK * 16;
  }
  // LDS offset of chunk idx
  __device__ static __forceinline__ int at(int idx) {
    if constexpr (KC) {
      const int r = idx >> 3, c = idx & 7;
      return r * 128 + ((c ^ ((r >> 1) & 7)) << 4);
    } else {
      const int k = idx / CPK, c = idx % CPK;
      if constexpr (ES == 2) {
        const int s = (k & 3) | (((k >> 3) & 1) << 2);
        return k * PITCH + (((c >> 1) ^ s) << 5) + ((c & 1) << 4);
      } else {
        return k * PITCH + (((c >> 2) ^ ((k >> 2) & 3)) << 6) + ((c & 3) << 4);
      }
    }
  }
  // Global loads of the K-tile at k0 (past ks: zeros).
  // kOdd: the dwords around a chunk, v and then x; store() shifts them.
  __device__ __forceinline__ void load(u32x4 (&v)[CH], unsigned (&x)[CH], int k0, int tid) const {
    if constexpr (BUF != kAny) {
      // from here to the last element of the tile's last row (KC) or k (KS)
      const long long from = KC ? (long long)k0 * ES : (long long)k0 * ld * ES;
      const long long bytes = (KC ? (long long)(rows - 1) * ld + ks : (long long)(ks - 1) * ld + rows) * ES - from;
      const char* base = p + from - odd;
      const u32x4 d = make_rsrc(base, (bytes + odd + 3) & ~3ll);  // (a dword that the end cuts counts as inside)
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((char*)base, 0, (int)d.z, 0x00020000);
      const int step = (int)(ld * ES) * (KC ? 32 : NT / CPK);  // bytes between a lane's chunks
      const int out = KC && (tid & 7) * EPC >= ks - k0 ? (int)0x80000000 : 0;  // k past the end of a row
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        int o = first + i * step;
        if constexpr (BUF == kOdd) {
          o = (o + odd) & ~3;
          // (the dword that holds the last element may hold the k after it too)
          if (!KC && k0 + (tid + i * NT) / CPK >= ks) o = (int)0x80000000;
        }
        v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o | out, 0, 0));
        if constexpr (BUF == kOdd) x[i] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rs, (o | out) + 16, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int idx = tid + i * NT;
        if constexpr (KC) {
          const int r = idx >> 3, k = k0 + (idx & 7) * EPC;
          v[i] = load_chunk<DT>(p + ((long long)r * ld + k) * ES, r < rows ? ks - k : 0);
        } else {
          const int k = k0 + idx / CPK, c = (idx % CPK) * EPC;
          v[i] = load_chunk<DT>(p + ((long long)k * ld + c) * ES, k < ks ? rows - c : 0);
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* lds, u32x4 (&v)[CH], const unsigned (&x)[CH], int k0, int tid) const {
    if constexpr (BUF == kOdd) {
      const int step = (int)(ld * ES) * (KC ? 32 : NT / CPK);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int by = ((first + odd + i * step) & 2) * 8;
        v[i] = u32x4{__builtin_amdgcn_alignbit(v[i][1], v[i][0], by), __builtin_amdgcn_alignbit(v[i][2], v[i][1], by),
                     __builtin_amdgcn_alignbit(v[i][3], v[i][2], by), __builtin_amdgcn_alignbit(x[i], v[i][3], by)};
      }
    }
    if (BUF != kAny && KC && ks % EPC && k0 + BK > ks) {  // the row ends inside 16 bytes: what follows it is not zero
#pragma unroll
      for (int i = 0; i < CH; ++i) v[i] = keep<DT>(v[i], ks - k0 - (tid & 7) * EPC);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int idx = tid + i * NT;
      if (R * 8 % NT == 0 || idx < R * 8) *(lds_u32x4_t*)(lds + at(idx)) = v[i];
    }
  }
  // Fragment half h (k 32 h .. + 31 in 16 bits, 16 h .. + 15 in fp32) of the
  // 16-row block at row r0: 16 bytes a lane.
  __device__ static __forceinline__ u32x4 frag(const char* lds, int r0, int h, int l16, int g) {
    if constexpr (KC) {
      const int r = r0 + l16;
      return *(const lds_u32x4_t*)(lds + r * 128 + (((4 * h + g) ^ ((r >> 1) & 7)) << 4));
    } else if constexpr (ES == 2) {
      const int q4 = l16 >> 2, p4 = l16 & 3, u = r0 >> 4;
      const char* q = lds + (32 * h + 8 * g + q4) * PITCH + ((u ^ (q4 | ((g & 1) << 2))) << 5) + p4 * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 4 * PITCH));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const char* q = lds + (16 * h + 4 * g) * PITCH + (((r0 >> 4) ^ g) << 6) + l16 * 4;
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *(const __attribute__((address_space(3))) unsigned*)(q + j * PITCH);
      return v;
    }
  }
};

// acc += one half K-tile (b first: a lane holds row l16, columns 4 g .. 4 g + 3).
template <int DT>
__device__ __forceinline__ void mma(f32x4& acc, const u32x4& b, const u32x4& a) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b[j]), __uint_as_float(a[j]), acc, 0, 0, 0);
  } else {
    acc = mfma16x16x32<DT>(__builtin_bit_cast(s16x8, b), __builtin_bit_cast(s16x8, a), acc);
  }
}

// RED: `reduce` (A and B are both KS). BM x BN tile, WR x 4 / WR waves; KW > 1: KW such
// sets of waves take every KW-th K-tile, and their sums meet in LDS, added in order.
template <int DT, bool RED, bool B_KC, int BM, int BN, int WR, int PF, int BUF, int KW>
__global__ void __launch_bounds__(NT * KW) gemm_grouped(GroupArgs a) {
  constexpr int ES = esize<DT>();
  using TA = Tile<DT, !RED, BM, BUF>;
  using TB = Tile<DT, B_KC, BN, BUF>;
  constexpr int BK = TA::BK;
  constexpr int WC = 4 / WR;
  constexpr int MB = BM / WR / 16, NB = BN / WC / 16;
  constexpr int STAGE = TA::BYTES + TB::BYTES;
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE * KW];

  const int tid = threadIdx.x % NT, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = KW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
  const int wr = w / WC, wc = w % WC, l16 = lane & 15, g = lane >> 4;

  const char *Ap, *Bp;
  char* Cp;
  int rows, cols, ks;  // of this tile: rows of C left, columns of C left, the sum's length
  if constexpr (RED) {
    const int per = a.tiles_m * a.tiles_n;
    const int e = blockIdx.x / per, t = blockIdx.x - e * per;
    const int m0 = t / a.tiles_n * BM, n0 = t % a.tiles_n * BN;
    const int r0 = __builtin_amdgcn_readfirstlane(group_end(a.ends, a.ends64, a.T, e - 1));
    const int r1 = __builtin_amdgcn_readfirstlane(group_end(a.ends, a.ends64, a.T, e));
    ks = r1 > r0 ? r1 - r0 : 0;
    rows = a.M - m0;
    cols = a.N - n0;
    Ap = (const char*)a.A + ((long long)r0 * a.lda + m0) * ES;
    Bp = (const char*)a.B + ((long long)r0 * a.ldb + n0) * ES;
    Cp = (char*)a.C + ((long long)e * a.sC + (long long)m0 * a.ldc + n0) * ES;
  } else {
    RowTile r;
    int tn;
    if (!find_tile<BM>(a, blockIdx.x, lane, r, tn)) return;
    const bool zero = r.e == a.E;
    ks = zero ? 0 : a.K;
    rows = r.rows;
    cols = a.N - tn * BN;
    Ap = (const char*)a.A + (long long)r.row0 * a.lda * ES;
    Bp = (const char*)a.B + ((long long)(zero ? 0 : r.e) * a.sB + (long long)tn * BN * (B_KC ? a.ldb : 1)) * ES;
    Cp = (char*)a.C + ((long long)r.row0 * a.ldc + (long long)tn * BN) * ES;
  }

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nk = (ks + BK - 1) / BK;
  if (nk > 0) {
    const TA ta(Ap, a.lda, rows, ks, tid);
    const TB tb(Bp, a.ldb, cols, ks, tid);
    u32x4 va[PF][TA::CH], vb[PF][TB::CH];
    unsigned xa[PF][TA::CH], xb[PF][TB::CH];
#pragma unroll
    for (int d = 0; d < PF; ++d) {
      ta.load(va[d], xa[d], (d * KW + kw) * BK, tid);
      tb.load(vb[d], xb[d], (d * KW + kw) * BK, tid);
    }
    for (int t0 = 0; t0 * KW < nk; t0 += PF) {
#pragma unroll
      for (int d = 0; d < PF; ++d) {
        const int t = t0 + d;  // K-tile t KW + kw (past the end: zeros)
        if (PF > 1 && t * KW >= nk) break;
        char* st = smem + (kw * 2 + (t & 1)) * STAGE;
        ta.store(st, va[d], xa[d], (t * KW + kw) * BK, tid);
        tb.store(st + TA::BYTES, vb[d], xb[d], (t * KW + kw) * BK, tid);
        ta.load(va[d], xa[d], ((t + PF) * KW + kw) * BK, tid);
        tb.load(vb[d], xb[d], ((t + PF) * KW + kw) * BK, tid);
        // this stage is written; the other one's readers are done (LDS only: loads stay in flight)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 fa[MB], fb[NB];
#pragma unroll
          for (int i = 0; i < MB; ++i) fa[i] = TA::frag(st, wr * (BM / WR) + i * 16, h, l16, g);
#pragma unroll
          for (int j = 0; j < NB; ++j) fb[j] = TB::frag(st + TA::BYTES, wc * (BN / WC) + j * 16, h, l16, g);
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) mma<DT>(acc[i][j], fb[j], fa[i]);
        }
      }
    }
  }

  if constexpr (KW > 1) {
    static_assert((KW - 1) * NT * MB * NB * 16 <= 2 * STAGE * KW, "the sums reuse the stages");
    float* red = (float*)smem + tid;
    __syncthreads();
    if (kw > 0) {
#pragma unroll
      for (int i = 0; i < MB * NB * 4; ++i)
        red[((kw - 1) * (MB * NB * 4) + i) * NT] = acc[i / (4 * NB)][i / 4 % NB][i % 4];
    }
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int i = 0; i < MB * NB * 4; ++i)
#pragma unroll
        for (int u = 0; u < KW - 1; ++u)
          acc[i / (4 * NB)][i / 4 % NB][i % 4] += red[(u * (MB * NB * 4) + i) * NT];
    }
    __syncthreads();
    if (kw > 0) return;
  }
  // Whole 16-byte pieces of C go out as rows through this wave's part of the LDS: stored
  // from the accumulators, a row's 32 bytes at a time, a weight gradient of 48 experts
  // of 167 rows, 2048 x 1024, takes 113 us instead of 80.
  constexpr int ROWB = NB * 16 * ES, PITCH = ROWB + 16, LPR = ROWB / 16, RPI = 64 / LPR;
  static_assert(4 * 16 * PITCH <= 2 * STAGE && 16 % RPI == 0 && 64 % (ROWB / 4) == 0, "epilogue rows");
  typedef __attribute__((address_space(3))) char lds_char;
  lds_char* eb = (lds_char*)(lds_void*)(smem + w * 16 * PITCH);
  const bool pieces = (uintptr_t)a.C % 16 == 0 && a.ldc * ES % 16 == 0 && a.sC * ES % 16 == 0 && a.N * ES % 16 == 0;
  const int col0 = wc * (BN / WC);
  if constexpr (KW == 1) __syncthreads();  // the last K-tile is read
#pragma unroll
  for (int i = 0; i < MB; ++i) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      lds_char* p = eb + l16 * PITCH + (j * 16 + 4 * g) * ES;
      if constexpr (DT == kF32) *(__attribute__((address_space(3))) f32x4*)p = acc[i][j];
      else *(lds_u32x2*)p = u32x2{pack2<DT>(acc[i][j][0], acc[i][j][1]), pack2<DT>(acc[i][j][2], acc[i][j][3])};
    }
    const int row0 = wr * (BM / WR) + i * 16;
    if (pieces) {
      const int rl = lane / LPR, cb = lane % LPR * 16;
      const bool in = col0 * ES + cb < cols * ES;
#pragma unroll
      for (int r = 0; r < 16 / RPI; ++r) {
        const u32x4 x = *(lds_u32x4_t*)(eb + (r * RPI + rl) * PITCH + cb);
        const int row = row0 + r * RPI + rl;
        if (in && row < rows) __builtin_nontemporal_store(x, (u32x4*)(Cp + row * a.ldc * ES + col0 * ES + cb));
      }
    } else {
      // Rows at any element: whole dwords of C, and the elements at a row's ends by themselves.
      constexpr int DPR = ROWB / 4, RPD = 64 / DPR;  // dwords a row, rows at once
      const int rl = lane / DPR, d = lane % DPR;
#pragma unroll
      for (int r = 0; r < 16 / RPD; ++r) {
        const int rr = r * RPD + rl, row = row0 + rr;
        if (row < rows) {
          char* q = Cp + (row * a.ldc + col0) * ES;
          if constexpr (ES == 4) {
            const unsigned x = *(const __attribute__((address_space(3))) unsigned*)(eb + rr * PITCH + 4 * d);
            if (col0 + d < cols) *(unsigned*)(q + 4 * d) = x;
          } else {
            typedef const __attribute__((address_space(3))) unsigned short lds_u16;
            const int off = (int)((uintptr_t)q >> 1) & 1, c = 2 * d + off;  // this lane's two columns
            const lds_u16* p = (const lds_u16*)(eb + rr * PITCH);
            const unsigned lo = p[c], hi = c + 1 < ROWB / 2 ? p[c + 1] : 0u;
            const int left = min(cols - col0, ROWB / 2) - c;
            if (left > 1) *(unsigned*)(q + 2 * c) = lo | hi << 16;
            if (left == 1) *(unsigned short*)(q + 2 * c) = (unsigned short)lo;
            if (off && d == 0 && cols > col0) *(unsigned short*)q = p[0];
          }
        }
      }
    }
  }
}

template <int DT, bool RED, bool B_KC, int BM, int BN, int WR, int PF, int KW = 1>
hipError_t launch(GroupArgs a, int buf, hipStream_t s) {
  a.tiles_m = (a.M + BM - 1) / BM;
  a.tiles_n = (a.N + BN - 1) / BN;
  const long long blocks = RED ? (long long)a.E * a.tiles_m * a.tiles_n
                               : (row_tiles_bound(a.T, a.E, BM, a.zero_tail) * a.tiles_n + 7) / 8 * 8;
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(NT * KW);
  if (buf == kDwords)
    hipLaunchKernelGGL((gemm_grouped<DT, RED, B_KC, BM, BN, WR, PF, kDwords, KW>), grid, block, 0, s, a);
  else if (DT != kF32 && buf == kOdd)
    hipLaunchKernelGGL((gemm_grouped<DT, RED, B_KC, BM, BN, WR, 1, DT == kF32 ? kAny : kOdd, KW>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((gemm_grouped<DT, RED, B_KC, BM, BN, WR, 1, kAny, KW>), grid, block, 0, s, a);
  return hipGetLastError();
}

// Row tiles of BM rows that T rows of E groups make, on average: every second
// group's last tile counts, and no group with rows goes without one.
inline double row_tiles(const GroupArgs& a, int bm) {
  const double t = (double)a.T / bm + 0.5 * a.E;
  const double least = a.T < a.E ? a.T : a.E;
  return t > least ? t : least;
}

// Microseconds of 64 k in 16 bits of `tiles` tiles: one where the CUs hold no second one, full
// where they hold `per` of them (measured: 256 x 256 tiles of grouped_w4.hip 1.5 us a
// round of 256; 128 x 128 alone 0.87, two a CU 1.83; 64 x 128 alone 0.6, three a CU 1.8).
// So 48 experts of 167 rows, 2048 x 1024, run on large tiles (58 us; 128 rows 80),
// of 43 rows on 64 (46; large ones 51), and 4 experts of 200 rows, where large tiles
// leave most CUs idle, on 64 as well (19; 128 rows 28, large ones 43).
inline double tile_time(double tiles, double alone, double full, int per) {
  if (tiles <= 256) return alone;
  const double t = full * tiles / (256.0 * per);
  return t > alone ? t : alone;
}
inline double large_time(double tiles) { return 1.5 * ceil(tiles / 256.0); }

template <int DT, bool B_KC>
hipError_t launch_rows(const GroupArgs& a, int buf, bool large, hipStream_t s) {
  // Rows a group has on average: a tile taller than that computes rows that
  // no group has, one shorter reads the weights once more for each tile.
  const int avg = (a.T + a.E - 1) / a.E;
  const int n128 = (a.N + 127) / 128;
  // Few tiles of a long sum: more waves of a tile share its K-tiles. (3 rows of 4 experts, 4096 x 2048:
  // one set of waves 32 us, 2 20, 4 18; 16 rows of 16, 4096 x 4096: 82, 82, 88; 25 rows of each of 4,
  // 2048 x 1024: 16.9, 12.5, 12.7.)
  const bool long_sum = a.K >= 16 * (DT == kF32 ? 32 : 64);
  const double few = row_tiles(a, avg <= 16 ? 16 : 32) * n128;
  if (avg <= 16) {
    if (long_sum && few <= 128) return launch<DT, false, B_KC, 16, 128, 1, 1, 4>(a, buf, s);
    if (long_sum && few <= 256) return launch<DT, false, B_KC, 16, 128, 1, 1, 2>(a, buf, s);
    return launch<DT, false, B_KC, 16, 128, 1, 1>(a, buf, s);
  }
  if constexpr (DT == kF32) {
    // an MFMA of 4 k takes as long as one of 32 in 16 bits: small tiles lose nothing to
    // loads, and pad groups and widths less (8 experts of 512 rows, 2048 x 2048: 32 x 64
    // 306 us, 64 x 64 315, 64 x 128 345, 128 x 128 402; 16 of 85, 1001 x 1416: 53, 60, 75)
    // few tiles, as above (621 rows of 9, 2048 x 256: 34 us alone, 24 in 4 sets; 800 of 6, 1536 x 512: 26, 20;
    // in 2 sets: 1150 of 4, 704 x 512 20, 18)
    const double t32 = row_tiles(a, 32) * ((a.N + 63) / 64);
    if (long_sum && t32 <= 160) return launch<DT, false, B_KC, 32, 64, 2, 2, 4>(a, buf, s);
    if (long_sum && t32 <= 320) return launch<DT, false, B_KC, 32, 64, 2, 2, 2>(a, buf, s);
    if (avg <= 256) return launch<DT, false, B_KC, 32, 64, 2, 2>(a, buf, s);
    return launch<DT, false, B_KC, 64, 64, 2, 2>(a, buf, s);
  } else {
    if (avg <= 32) {
      if (long_sum && few <= 256) return launch<DT, false, B_KC, 32, 128, 1, 1, 2>(a, buf, s);
      return launch<DT, false, B_KC, 32, 128, 1, 1>(a, buf, s);
    }
    const int n256 = (a.N + 255) / 256;
    const double t64 = tile_time(row_tiles(a, 64) * n128, 0.6, 1.8, 3);
    const double t128 = tile_time(row_tiles(a, 128) * n128, 0.87, 1.83, 2);
    if (large && large_time(row_tiles(a, 256) * n256) <= (t64 < t128 ? t64 : t128))
      return grouped_w4(a, DT, false, B_KC, s);
    // few tiles again (1000 rows of 4, 4096 x 512: 64 rows a tile 37 us, in 2 sets 27, 32 rows in 4 sets 20; 529
    // of 6, 2496 x 1344: 22.8, 19.3, 15.5; 150 of 4, 1024 x 2048: 11.8, -, 8.7)
    if (long_sum && row_tiles(a, 32) * n128 <= 256) return launch<DT, false, B_KC, 32, 128, 1, 1, 4>(a, buf, s);
    if (long_sum && row_tiles(a, 64) * n128 <= 256) return launch<DT, false, B_KC, 64, 128, 2, 1, 2>(a, buf, s);
    if (t64 < t128) return launch<DT, false, B_KC, 64, 128, 2, 1>(a, buf, s);
    return launch<DT, false, B_KC, 128, 128, 2, 1>(a, buf, s);
  }
}

template <int DT>
hipError_t launch_reduce(const GroupArgs& a, int buf, bool large, hipStream_t s) {
  if constexpr (DT == kF32) {
    // (2048 rows of 4, 256 x 512: one set of waves 15.0 us, 2 13.5; 4096 of 8: 15.8, 14.7)
    if (a.T >= 256ll * a.E && (double)a.E * ((a.M + 63) / 64) * ((a.N + 63) / 64) <= 256)
      return launch<DT, true, false, 64, 64, 2, 2, 2>(a, buf, s);
    return launch<DT, true, false, 64, 64, 2, 2>(a, buf, s);
  } else {
    // As above, with what a tile costs beside its 64-k steps: large ones 5 us, 128 x 128
    // 1.5 (3 alone). (48 experts of 167 rows, 2048 x 1024: large 66 us, 128 rows 80; 64 experts of
    // 32 rows: 82, 60; 16 of 512: 43, 58.)
    const double nk = ((double)a.T / a.E + 63) / 64, even = nk < 4 ? 4 : nk + 1;
    const double t256 = (double)a.E * ((a.M + 255) / 256) * ((a.N + 255) / 256);
    const double t128 = (double)a.E * ((a.M + 127) / 128) * ((a.N + 127) / 128);
    const double small = t128 <= 256 ? 0.87 * nk + 3 : (1.83 * nk + 1.5) * (t128 <= 512 ? 1.0 : t128 / 512);
    if (large && (1.5 * even + 5) * ceil(t256 / 256) <= small) return grouped_w4(a, DT, true, false, s);
    // (4096 rows of 4, 512 x 512: one set of waves 16.6 us, 2 14.6; 8192 of 4, 1024 x 1024: 30.5, 27.3; but
    // 4096 of 8, 512 x 768: 11.8, 12.9)
    if (nk >= 12 && t128 <= 256) return launch<DT, true, false, 128, 128, 2, 1, 2>(a, buf, s);
    return launch<DT, true, false, 128, 128, 2, 1>(a, buf, s);
  }
}

}  // namespace kgrp

// Buffer loads take any multiple of 4 bytes; their offsets stay below 2^31 in 128
// rows (KC) or 64 k (KS) of an operand.
static int loads_of(const void* p, long long ld, long long batch, int es) {
  if (ld * es > (1ll << 23)) return kgrp::kAny;
  return (uintptr_t)p % 4 == 0 && ld * es % 4 == 0 && batch * es % 4 == 0 ? kgrp::kDwords : kgrp::kOdd;
}

hipError_t grouped_gemm(const GroupedProblem& p, hipStream_t stream) {
  const int es = p.dtype == kF32 ? 4 : 2;
  const bool red = p.kind == kGroupReduce;
  // nothing to compute or to write
  if (p.N == 0 || p.E == 0 || (red ? p.M == 0 : p.T == 0)) return hipSuccess;
  GroupArgs a{};
  a.A = p.A;
  a.B = p.B;
  a.C = p.C;
  a.ends = p.ends;
  a.ends64 = p.ends64;
  a.E = p.E;
  a.T = p.T;
  a.M = p.M;
  a.N = p.N;
  a.K = p.K;
  a.lda = p.lda;
  a.ldb = p.ldb;
  a.ldc = p.ldc;
  a.sB = p.sB;
  a.sC = p.sC;
  a.zero_tail = p.zero_tail;
  const int la = loads_of(p.A, p.lda, 0, es), lb = loads_of(p.B, p.ldb, p.sB, es);
  const int buf = la == kgrp::kAny || lb == kgrp::kAny ? kgrp::kAny : la == lb ? la : kgrp::kOdd;
  const bool large = p.dtype != kF32 && grouped_w4_ok(a, red, p.b_colmajor);
  switch (p.dtype) {
    case kF32:
      return red            ? kgrp::launch_reduce<kF32>(a, buf, large, stream)
             : p.b_colmajor ? kgrp::launch_rows<kF32, true>(a, buf, large, stream)
                            : kgrp::launch_rows<kF32, false>(a, buf, large, stream);
    case kF16:
      return red            ? kgrp::launch_reduce<kF16>(a, buf, large, stream)
             : p.b_colmajor ? kgrp::launch_rows<kF16, true>(a, buf, large, stream)
                            : kgrp::launch_rows<kF16, false>(a, buf, large, stream);
    case kBF16:
      return red            ? kgrp::launch_reduce<kBF16>(a, buf, large, stream)
             : p.b_colmajor ? kgrp::launch_rows<kBF16, true>(a, buf, large, stream)
                            : kgrp::launch_rows<kBF16, false>(a, buf, large, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace pdmb
