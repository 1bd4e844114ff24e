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
// This kernel stages global -> registers -> LDS, so that any alignment and any
// size is right: chunks past an edge are zero, chunks that an edge cuts are read by
// the element. Two LDS stages, one barrier a K-tile, the next K-tile's loads in
// flight during a K-tile's MFMAs.
#include "api.h"
#include "grouped.h"

namespace pdmb {
namespace kgrp {

constexpr int NT = 256;

template <int DT>
constexpr int esize() { return DT == kF32 ? 4 : 2; }

// 16 bytes at p, of which `avail` elements are inside the operand. VEC: p is
// 16-B aligned and an edge never cuts a chunk.
template <int DT, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const char* p, int avail) {
  constexpr int ES = esize<DT>(), EPC = 16 / ES;
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (avail > 0) v = *(const u32x4*)p;
  } else if (avail >= EPC) {
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

// One operand tile of R rows (or columns) x one K-tile.
template <int DT, bool KC, int R>
struct Tile {
  static constexpr int ES = esize<DT>(), EPC = 16 / ES, BK = 128 / ES;
  static constexpr int BYTES = R * 128;
  static constexpr int CH = (R * 8 + NT - 1) / NT;  // chunks a thread
  static constexpr int PITCH = R * ES;              // KS image: bytes of one k
  static_assert(KC || R >= 128, "KS swizzle spans 8 units");

  // LDS offset of chunk idx
  __device__ static __forceinline__ int at(int idx) {
    if constexpr (KC) {
      const int r = idx >> 3, c = idx & 7;
      return r * 128 + ((c ^ ((r >> 1) & 7)) << 4);
    } else {
      constexpr int CPK = PITCH / 16;
      const int k = idx / CPK, c = idx % CPK;
      if constexpr (ES == 2) {
        const int s = (k & 3) | (((k >> 3) & 1) << 2);
        return k * PITCH + (((c >> 1) ^ s) << 5) + ((c & 1) << 4);
      } else {
        return k * PITCH + (((c >> 2) ^ ((k >> 2) & 3)) << 6) + ((c & 3) << 4);
      }
    }
  }
  // Global loads of K-tile at k0: p is the operand at its first row / column
  // and k = 0, ld its leading stride, `rows` and `ks` what is left of it.
  template <bool VEC>
  __device__ static __forceinline__ void load(u32x4 (&v)[CH], const char* p, long long ld, int rows, int k0, int ks,
                                              int tid) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int idx = tid + i * NT;
      if constexpr (KC) {
        const int r = idx >> 3, k = k0 + (idx & 7) * EPC;
        v[i] = load_chunk<DT, VEC>(p + ((long long)r * ld + k) * ES, r < rows ? ks - k : 0);
      } else {
        constexpr int CPK = PITCH / 16;
        const int k = k0 + idx / CPK, c = (idx % CPK) * EPC;
        v[i] = load_chunk<DT, VEC>(p + ((long long)k * ld + c) * ES, k < ks ? rows - c : 0);
      }
    }
  }
  __device__ static __forceinline__ void store(char* lds, const u32x4 (&v)[CH], int tid) {
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
      const char* p = lds + (32 * h + 8 * g + q4) * PITCH + ((u ^ (q4 | ((g & 1) << 2))) << 5) + p4 * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * PITCH));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const char* p = lds + (16 * h + 4 * g) * PITCH + (((r0 >> 4) ^ g) << 6) + l16 * 4;
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *(const __attribute__((address_space(3))) unsigned*)(p + j * PITCH);
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

// Four columns of one row, `left` of them inside C. ALIGNED: 4 elements at once.
template <int DT, bool ALIGNED>
__device__ __forceinline__ void store4(char* p, const f32x4& v, int left) {
  if constexpr (DT == kF32) {
    if (ALIGNED && left >= 4) {
      *(f32x4*)p = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) ((float*)p)[j] = v[j];
    }
  } else {
    const u32x2 w = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    if (ALIGNED && left >= 4) {
      *(u32x2*)p = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) ((unsigned short*)p)[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// RED: `reduce` (A and B are both KS). BM x 128 tile, 4 waves: 2 x 2 for BM >=
// 64, else 1 x 4. VEC: 16-B aligned operands whose edges fall between chunks,
// and a C that takes 4 elements at once.
template <int DT, bool RED, bool B_KC, int BM, bool VEC>
__global__ void __launch_bounds__(NT) grouped(GroupArgs a) {
  constexpr int BN = 128, ES = esize<DT>();
  using TA = Tile<DT, !RED, BM>;
  using TB = Tile<DT, B_KC, BN>;
  constexpr int BK = TA::BK;
  constexpr int WR = BM >= 64 ? 2 : 1, WC = 4 / WR;
  constexpr int MB = BM / WR / 16, NB = BN / WC / 16;
  constexpr int STAGE = TA::BYTES + TB::BYTES;
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = w / WC, wc = w % WC, l16 = lane & 15, g = lane >> 4;

  const char *Ap, *Bp;
  char* Cp;
  int rows, cols, ks;  // of this tile: rows of C left, columns of C left, the sum's length
  bool zero = false;
  if constexpr (RED) {
    const int per = a.tiles_m * a.tiles_n;
    const int e = blockIdx.x / per, t = blockIdx.x - e * per;
    const int m0 = t / a.tiles_n * BM, n0 = t % a.tiles_n * BN;
    const int r0 = group_end(a.ends, a.ends64, a.T, e - 1), r1 = group_end(a.ends, a.ends64, a.T, e);
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
    zero = r.e == a.E;
    ks = zero ? 0 : a.K;
    rows = r.rows;
    cols = a.N - tn * BN;
    Ap = (const char*)a.A + (long long)r.row0 * a.lda * ES;
    Bp = (const char*)a.B + ((long long)(zero ? 0 : r.e) * a.sB + (long long)tn * BN * (B_KC ? a.ldb : 1)) * ES;
    Cp = (char*)a.C + ((long long)r.row0 * a.ldc + tn * BN) * ES;
  }

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nk = (ks + BK - 1) / BK;
  u32x4 va[TA::CH], vb[TB::CH];
  if (nk > 0) {
    TA::template load<VEC>(va, Ap, a.lda, rows, 0, ks, tid);
    TB::template load<VEC>(vb, Bp, a.ldb, cols, 0, ks, tid);
  }
  for (int t = 0; t < nk; ++t) {
    char* st = smem + (t & 1) * STAGE;
    TA::store(st, va, tid);
    TB::store(st + TA::BYTES, vb, tid);
    if (t + 1 < nk) {
      TA::template load<VEC>(va, Ap, a.lda, rows, (t + 1) * BK, ks, tid);
      TB::template load<VEC>(vb, Bp, a.ldb, cols, (t + 1) * BK, ks, tid);
    }
    __syncthreads();  // this stage is written; the other one's readers are done
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

#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int r = wr * (BM / WR) + i * 16 + l16;
    if (r < rows) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int c = wc * (BN / WC) + j * 16 + 4 * g;
        store4<DT, VEC>(Cp + ((long long)r * a.ldc + c) * ES, acc[i][j], cols - c);
      }
    }
  }
}

template <int DT, bool RED, bool B_KC, int BM>
hipError_t launch(const GroupArgs& a, bool vec, unsigned grid, hipStream_t s) {
  if (vec)
    hipLaunchKernelGGL((grouped<DT, RED, B_KC, BM, true>), dim3(grid), dim3(NT), 0, s, a);
  else
    hipLaunchKernelGGL((grouped<DT, RED, B_KC, BM, false>), dim3(grid), dim3(NT), 0, s, a);
  return hipGetLastError();
}

template <int DT, bool B_KC>
hipError_t launch_rows(GroupArgs a, bool vec, hipStream_t s) {
  // Rows a group has on average: a tile taller than that computes rows that
  // no group has, one shorter reads the weights once more for each tile.
  const int avg = (a.T + a.E - 1) / a.E;
  const int bm = avg <= 16 ? 16 : avg <= 32 ? 32 : avg <= 64 ? 64 : 128;
  a.tiles_n = (a.N + 127) / 128;
  const long long prods = row_tiles_bound(a.T, a.E, bm, a.zero_tail) * a.tiles_n;
  if (prods > (1ll << 30)) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)((prods + 7) / 8 * 8);
  switch (bm) {
    case 16: return launch<DT, false, B_KC, 16>(a, vec, grid, s);
    case 32: return launch<DT, false, B_KC, 32>(a, vec, grid, s);
    case 64: return launch<DT, false, B_KC, 64>(a, vec, grid, s);
    default: return launch<DT, false, B_KC, 128>(a, vec, grid, s);
  }
}

template <int DT>
hipError_t launch_reduce(GroupArgs a, bool vec, hipStream_t s) {
  a.tiles_m = (a.M + 127) / 128;
  a.tiles_n = (a.N + 127) / 128;
  const long long blocks = (long long)a.E * a.tiles_m * a.tiles_n;
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  return launch<DT, true, false, 128>(a, vec, (unsigned)blocks, s);
}

}  // namespace kgrp

static bool vec_ok(const void* p, long long ld, long long batch, int es, int edge) {
  const int epc = 16 / es;
  return (uintptr_t)p % 16 == 0 && ld % epc == 0 && batch % epc == 0 && edge % epc == 0;
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
  const bool c_ok = (uintptr_t)p.C % (4 * es) == 0 && p.ldc % 4 == 0 && p.sC % 4 == 0;
  const bool vec = c_ok && vec_ok(p.A, p.lda, 0, es, red ? p.M : p.K) &&
                   vec_ok(p.B, p.ldb, p.sB, es, red || !p.b_colmajor ? p.N : p.K);
  const int avg = (p.T + p.E - 1) / p.E;
  if (p.dtype != kF32 && (red ? p.M >= 256 && p.N >= 256 : avg >= 192) && (red || p.K > 0) &&
      grouped_w4_ok(a, red, p.b_colmajor))
    return grouped_w4(a, p.dtype, red, p.b_colmajor, stream);
  switch (p.dtype) {
    case kF32:
      return red            ? kgrp::launch_reduce<kF32>(a, vec, stream)
             : p.b_colmajor ? kgrp::launch_rows<kF32, true>(a, vec, stream)
                            : kgrp::launch_rows<kF32, false>(a, vec, stream);
    case kF16:
      return red            ? kgrp::launch_reduce<kF16>(a, vec, stream)
             : p.b_colmajor ? kgrp::launch_rows<kF16, true>(a, vec, stream)
                            : kgrp::launch_rows<kF16, false>(a, vec, stream);
    case kBF16:
      return red            ? kgrp::launch_reduce<kBF16>(a, vec, stream)
             : p.b_colmajor ? kgrp::launch_rows<kBF16, true>(a, vec, stream)
                            : kgrp::launch_rows<kBF16, false>(a, vec, stream);
    default:
      return hipErrorInvalidValue;
  }
}

}  // namespace pdmb
