// int4.hip — products of a few rows with 4-bit weights and group scales:
//   C[r][n] = sum over groups j of scale[n][j] * sum over k in group j of X[r][k] (q[n][k] - zero[n][j])
// for bf16 / fp16 rows, one weight or (grouped by expert) one for each group
// of rows.
//
// Exactness: the nibbles go into the matrix instructions as whole numbers, so
// a weight is never rounded. Two values at a time, at one place of a dword's
// halves, become B + q (a power of two B whose mantissa step fits the place) by
// one and-or, most after one shift:
//   bf16  B = 16: every nibble shifted to bits 3-6
//   fp16  B = 1024: nibbles 0 and 2 at bits 0-3, 1 and 3 at bits 4-7 (16 times the value)
// fp16 then subtracts B + zero exactly (v_pk_add_f16, for bits 4-7 v_pk_fma_f16 with
// 1/16); bf16, which has no packed add, adds a second product with the constants
// -(16 + zero), also whole numbers, to the same fp32 sum. Each group's fp32 sum is
// scaled once, in fp32.
//
// So a bf16 sum's terms are x (16 + q) and -x (16 + zero), not x (q - zero): its fp32 error is relative to
// |x| (32 + q + zero) (B = 128 for nibble 0, which needs no shift, is one instruction a dword less and
// made that up to eight times as much), a row whose 31 sum |x| over a group passes 3.4e38 gives NaN, and so
// does a row with an infinity: the two products cancel.
//
// Loads: an MFMA operand has its 16 columns in neighbouring lanes, but 16-byte
// loads whose neighbours are in 16 rows of memory look a cache line up for
// every lane (measured: 13 bytes a ns and CU whatever the tile, depth or number of
// waves). So four lanes load 64 bytes of one column, 128 k, and
// ds_bpermute brings each dword to the operand's lane (l16, g): 16 bytes, k 32 g ..
// + 31. Its four dwords are then transposed among the four 16-lane rows (two
// v_permlane32_swap, two v_permlane16_swap): dword j holds k 32 j + 8 g .. + 7,
// and MFMA j covers 32 consecutive k, the smallest group. A dword's halves hold
// nibbles i and i + 4; the rows' fragments are permuted the same way on their way
// through LDS ([row][256 B], 16-B piece c at c ^ row: conflict-free both ways).
//
// Two kernels: gemm_int4_few for 16 rows a tile and short sums or narrow weights, and
// gemm_int4_rows for more, where the rows of a block come through LDS once for 64 columns.
// What bounds them: 1 row, 8192 x 16384: 14.9 us, the read of the weight (4.6 TB/s) with 7 us of
// widening beside it; 16 rows, 4096 x 11007, groups of 32: 11.4 us, of which the vector
// units work 5.0 (34 instructions for an MFMA) and the rest is launch, first loads and the
// join; 100 rows, 4096 x 8192: 21.8 us, vector units 9.7, matrix units 7 (two products for
// a bf16 weight) and LDS 5, which overlap little with a barrier a step.
#include "api.h"
#include "grouped.h"

namespace pdmb {
namespace kint4 {

struct Args : GroupArgs {
  const void* scale;
  const unsigned char* zero;
  int groups;   // K / G
  long long scales;  // E N groups
  unsigned chunk_g;  // G > 128: ceil(2^32 / (G / 128)), else 0
};

// Group of chunk c where a group is one chunk or more. (c and G / 128 are at most K / 128
// <= 2^16, so the product with the rounded-up reciprocal is exact.)
__device__ __forceinline__ int group_of(const Args& a, int c) {
  return a.chunk_g ? (int)__umulhi((unsigned)c, a.chunk_g) : c;
}

// {r0, r1, r2, r3} of lane row g -> dword g of lane rows 0 .. 3
__device__ __forceinline__ void transpose4(u32x4& r) {
  auto a = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  r = u32x4{c[0], c[1], d[0], d[1]};
}

// x0 .. x7 -> (x0, x4), (x1, x5), (x2, x6), (x3, x7)
__device__ __forceinline__ s16x8 permute_row(const u32x4& x) {
  const u32x4 v = {__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                   __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
  return __builtin_bit_cast(s16x8, v);
}

// The and-or constants in registers (an instruction that does both takes no literal).
struct Bits {
  unsigned mask0, mask1, or0, or1;
  template <int DT>
  __device__ static __forceinline__ Bits make() {
    Bits b = DT == kBF16 ? Bits{0u, 0x00780078u, 0u, 0x41804180u}
                         : Bits{0x000f000fu, 0x00f000f0u, 0x64006400u, 0x64006400u};
    asm("" : "+s"(b.mask1), "+v"(b.or1));
    if constexpr (DT != kBF16) asm("" : "+s"(b.mask0), "+v"(b.or0));
    return b;
  }
};

// What widen() subtracts for a zero point, two halves each. bf16: -(16 + zero). fp16: [0] -(B + zero) of the
// first pair, [1] of the others -(64 + zero), after the 1/16.
struct Minus {
  unsigned m[2];
};
template <int DT>
__device__ __forceinline__ Minus minus_of(unsigned z) {
  // (bf16 16 + z: step 1 at bit 3; fp16 1024 + z: bit 0, 64 + z: bit 4)
  return DT == kBF16 ? Minus{{z * 0x00080008u + 0xc180c180u, z * 0x00080008u + 0xc180c180u}}
                     : Minus{{z * 0x00010001u + 0xe400e400u, z * 0x00100010u + 0xd400d400u}};
}

// 8 nibbles as B + q (bf16), or as q - zero (fp16).
template <int DT>
__device__ __forceinline__ s16x8 widen(unsigned d, const Bits& b, const Minus& minus) {
  u32x4 v;
  if constexpr (DT == kBF16) {
    v = u32x4{((d << 3) & b.mask1) | b.or1, ((d >> 1) & b.mask1) | b.or1, ((d >> 5) & b.mask1) | b.or1,
              ((d >> 9) & b.mask1) | b.or1};
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 m0 = __builtin_bit_cast(f16x2, minus.m[0]), m1 = __builtin_bit_cast(f16x2, minus.m[1]);
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned e = d >> 8;
    const f16x2 w[4] = {__builtin_bit_cast(f16x2, (d & b.mask0) | b.or0) + m0,
                        __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (d & b.mask1) | b.or1), sixteenth, m1),
                        __builtin_bit_cast(f16x2, (e & b.mask0) | b.or0) + m0,
                        __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (e & b.mask1) | b.or1), sixteenth, m1)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, w[i]);
  }
  return __builtin_bit_cast(s16x8, v);
}

// A chunk of 128 k has SG scales and zero points of a column: G = 32: 4, 64: 2, 128 and
// more: 1. ZERO: zero points are given (otherwise 8).
template <int SG, int DT, bool ZERO>
struct Scales {
  unsigned s[(SG + 1) / 2], z;
  __device__ __forceinline__ void load_lds(const char* sp, const char* zp) {
    typedef __attribute__((address_space(3))) unsigned lds_u32;
    typedef __attribute__((address_space(3))) unsigned short lds_u16;
    typedef __attribute__((address_space(3))) unsigned char lds_u8;
    if constexpr (SG == 1) {
      s[0] = *(const lds_u16*)sp;
      if constexpr (ZERO) z = *(const lds_u8*)zp;
    } else if constexpr (SG == 2) {
      s[0] = *(const lds_u32*)sp;
      if constexpr (ZERO) z = *(const lds_u16*)zp;
    } else {
      const u32x2 v = *(const lds_u32x2*)sp;
      s[0] = v.x;
      s[1] = v.y;
      if constexpr (ZERO) z = *(const lds_u32*)zp;
    }
  }
  __device__ __forceinline__ float scale(int t) const {
    if constexpr (DT == kBF16) return __uint_as_float(t & 1 ? s[t >> 1] & 0xffff0000u : s[t >> 1] << 16);
    else return to_f32<DT>((unsigned short)(s[t >> 1] >> (16 * (t & 1))));
  }
  __device__ __forceinline__ unsigned zero(int t) const { return ZERO ? (z >> (8 * t)) & 15u : 8u; }
};

// Scales and zero points of COLS columns and KB chunks go to LDS before they are
// used, 8 groups a lane: read where they are used they cost a cache line look-up for
// every lane (a 16 x 4096 x 11007 product with groups of 32: 128 of a chunk's 208).
// [column][KB * SG groups], 8 bytes between columns against bank conflicts.
template <int DT, int COLS, int SG, int KB, bool ZERO, int THREADS>
struct ScaleBlock {
  static constexpr int NG = KB * SG, SP = 2 * NG + 8, ZP = NG + 8, BYTES = COLS * (SP + ZP);
  static constexpr int CHUNKS = KB, PIECES = COLS * NG / 8, CH = (PIECES + THREADS - 1) / THREADS;
  u32x4 s[CH];
  u32x2 z[CH];
  int back[CH];  // groups the load was moved back by, not to pass the array's end
  // groups from g0 of columns from n0 (of expert e's `first`); what is not there is stored as zero
  __device__ __forceinline__ void load(const Args& a, long long first, int n0, int g0, int tid) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = tid + i * THREADS, col = at / (NG / 8), gr = g0 + at % (NG / 8) * 8;
      const long long off = (first + min(n0 + col, a.N - 1)) * a.groups + gr;
      // (no branch around these loads: each would wait for its own)
      const long long at8 = off < a.scales - 8 ? off : a.scales < 8 ? 0 : a.scales - 8;
      const unsigned short* sp = (const unsigned short*)a.scale + at8;
      const unsigned char* zp = a.zero + at8;
      u32x4 v;
      u32x2 w = {0u, 0u};
      if (a.scales >= 8) {
        __builtin_memcpy(&v, sp, 16);
        if constexpr (ZERO) __builtin_memcpy(&w, zp, 8);
      } else {  // (fewer in all: each by itself, the last one again past the end)
        const int n = (int)a.scales - 1;
        auto pair = [&](int t) { return (unsigned)sp[min(t, n)] | (unsigned)sp[min(t + 1, n)] << 16; };
        v = u32x4{pair(0), pair(2), pair(4), pair(6)};
        auto four = [&](int t) {
          return (unsigned)zp[min(t, n)] | (unsigned)zp[min(t + 1, n)] << 8 | (unsigned)zp[min(t + 2, n)] << 16 |
                 (unsigned)zp[min(t + 3, n)] << 24;
        };
        if constexpr (ZERO) w = u32x2{four(0), four(4)};
      }
      s[i] = v;
      z[i] = w;
      back[i] = (int)(off - at8);
    }
  }
  __device__ __forceinline__ void store(const Args& a, char* lds, int g0, int tid) const {
    typedef unsigned long long u64;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = tid + i * THREADS, col = at / (NG / 8), gr = at % (NG / 8) * 8;
      u64 lo = (u64)s[i][1] << 32 | s[i][0], hi = (u64)s[i][3] << 32 | s[i][2], zz = 0;
      if constexpr (ZERO) zz = (u64)z[i].y << 32 | z[i].x;
      const int left = a.groups - g0 - gr;  // groups from here to the column's last
      if (left < 8) {
        const int b = min(back[i], 8);
        lo = b >= 8 ? 0 : b >= 4 ? hi >> (16 * (b - 4)) : b ? lo >> (16 * b) | hi << (64 - 16 * b) : lo;
        hi = b >= 4 ? 0 : hi >> (16 * b);
        zz = b >= 8 ? 0 : zz >> (8 * b);
        if (left < 4) lo = left <= 0 ? 0 : lo & ((1ull << (16 * left)) - 1);
        hi = left <= 4 ? 0 : hi & ((1ull << (16 * (left - 4))) - 1);
        zz = left <= 0 ? 0 : zz & ((1ull << (8 * left)) - 1);
      }
      if (PIECES % THREADS == 0 || at < PIECES) {
        char* p = lds + col * SP + 2 * gr;
        *(lds_u32x2*)p = u32x2{(unsigned)lo, (unsigned)(lo >> 32)};
        *(lds_u32x2*)(p + 8) = u32x2{(unsigned)hi, (unsigned)(hi >> 32)};
        if constexpr (ZERO) *(lds_u32x2*)(lds + COLS * SP + col * ZP + gr) = u32x2{(unsigned)zz, (unsigned)(zz >> 32)};
      }
    }
  }
  // column c, SG groups from `at` of the block
  __device__ static __forceinline__ void read(Scales<SG, DT, ZERO>& v, const char* lds, int c, int at) {
    v.load_lds(lds + c * SP + 2 * at, lds + COLS * SP + c * ZP + at);
  }
};

// Where a lane loads of column block j: column 16 j + (lane >> 2), 16-byte piece lane & 3.
template <int NB>
struct Weights {
  const unsigned char* p[NB];
  int tail;  // moves the piece inside a partial last chunk (any weight will do: the rows are zero there)
  __device__ __forceinline__ Weights(const Args& a, long long first, int n0, int lane) {
    const int piece = 16 * (lane & 3), part = a.K % 128;
#pragma unroll
    for (int j = 0; j < NB; ++j)
      p[j] = (const unsigned char*)a.B + (first + min(n0 + 16 * j + (lane >> 2), a.N - 1)) * (a.K / 2) + piece;
    tail = part ? min(piece, part / 2 - 16) - piece : 0;
  }
  // chunk c of nc (past the end: the last one again)
  __device__ __forceinline__ void load(u32x4 (&q)[NB], int c, int nc) const {
    c = min(c, nc - 1);
    const int at = c * 64 + (c == nc - 1 ? tail : 0);
#pragma unroll
    for (int j = 0; j < NB; ++j) q[j] = *(const u32x4*)(p[j] + at);
  }
};

// As loaded -> the operand's lanes (column l16, k 32 j + 8 g .. + 7 in dword j).
__device__ __forceinline__ void to_operand(u32x4& v, int from) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (unsigned)__builtin_amdgcn_ds_bpermute(from, (int)v[i]);
  transpose4(v);
}

// The tile's rows as a buffer whose range ends with the last row: offsets of
// rows (or k) that there are not go past it and read as zeros, with no branch.
constexpr int kOutside = (int)0x80000000;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const Args& a, const RowTile& r) {
  return __builtin_amdgcn_make_buffer_rsrc((char*)a.A + (long long)r.row0 * a.lda * 2, 0,
                                           (int)(((long long)(r.rows - 1) * a.lda + a.K) * 2), 0x00020000);
}
__device__ __forceinline__ u32x4 load_row(__amdgpu_buffer_rsrc_t x, int off, int soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(x, off, soff, 0));
}

// ---- up to 16 rows -------------------------------------------------------
// A workgroup takes 16 NB columns, its W waves a run of k each, one chunk of 128 k a
// step with the next D in flight; each wave passes its part of the rows (4 RX
// of them) through LDS of its own. The W sums meet in LDS, added in wave order.
//
// The loop has no branches around loads (a conditional load makes hipcc wait for
// the loads after it as well): chunk numbers past the end repeat the last one and
// are not computed; a partial last chunk reads weights from inside the column
// and zeros for the rows.

template <int NB, int RX>
struct Step {
  u32x4 q[NB], x[RX];
};

template <int DT, int NB, int SG, int RX, bool ZERO, class SB>
__device__ __forceinline__ void multiply(f32x4 (&acc)[NB], Step<NB, RX>& b, const Bits& bits, char* xl, const char* sl,
                                         int at, int lane) {
  constexpr int PER = 4 / SG;  // MFMAs of a group
  const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < RX; ++i) {
    const int row = 4 * i + g;  // piece l16 of it
    *(lds_u32x4_t*)(xl + row * 256 + ((l16 ^ row) << 4)) = __builtin_bit_cast(u32x4, permute_row(b.x[i]));
  }
  Scales<SG, DT, ZERO> sc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    SB::read(sc[j], sl, 16 * j + l16, at);
    to_operand(b.q[j], (l16 * 4 + g) * 4);
  }
  f32x4 p[NB];
  Minus minus[NB];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const s16x8 xf = *(const lds_s16x8*)(xl + l16 * 256 + (((4 * t + g) ^ l16) << 4));
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (t % PER == 0) {
        minus[j] = minus_of<DT>(sc[j].zero(t / PER));
        p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      p[j] = mfma16x16x32<DT>(xf, widen<DT>(b.q[j][t], bits, minus[j]), p[j]);
      if constexpr (DT == kBF16) {
        const u32x4 m = {minus[j].m[0], minus[j].m[1], minus[j].m[1], minus[j].m[1]};
        p[j] = mfma16x16x32<DT>(xf, __builtin_bit_cast(s16x8, m), p[j]);
      }
    }
    if (t % PER == PER - 1) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float s = sc[j].scale(t / PER);
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[j][v] = fmaf(s, p[j][v], acc[j][v]);
      }
    }
  }
}

// The wave's part of a tile's sums: 16 NB columns from n0, its run of k.
template <int DT, int NB, int SG, int RX, bool ZERO, int W, int D, class SB>
__device__ __forceinline__ void few_sums(const Args& a, const RowTile& r, int n0, int tid, int w, char* xl, char* sl,
                                         f32x4 (&acc)[NB]) {
  const int lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int nc = r.e == a.E ? 0 : (a.K + 127) / 128;  // (rows behind the last group: zeros)
  if (nc > 0) {
    const int part = a.K % 128;  // k of a partial last chunk
    const long long first = (long long)r.e * a.N;
    const Weights<NB> q(a, first, n0, lane);
    const __amdgpu_buffer_rsrc_t xr = rows_buffer(a, r);
    int xo[RX], xt[RX];  // row offsets, and those of the last chunk
#pragma unroll
    for (int i = 0; i < RX; ++i) {
      xo[i] = 4 * i + g < r.rows ? (4 * i + g) * (int)a.lda * 2 + 16 * l16 : kOutside;
      xt[i] = part && 8 * l16 >= part ? kOutside : xo[i];
    }
#pragma unroll
    for (int i = RX * 4 + g; i < 16; i += 4)  // rows that there are not
      *(lds_u32x4_t*)(xl + i * 256 + (l16 << 4)) = u32x4{0u, 0u, 0u, 0u};
    const Bits bits = Bits::make<DT>();

    auto load = [&](Step<NB, RX>& b, int c) {
      q.load(b.q, c, nc);
      c = min(c, nc - 1);
#pragma unroll
      for (int i = 0; i < RX; ++i) b.x[i] = load_row(xr, c == nc - 1 ? xt[i] : xo[i], c * 256);
    };

    for (int k0 = 0; k0 < nc; k0 += SB::CHUNKS) {
      const int kn = min(SB::CHUNKS, nc - k0), per = (kn + W - 1) / W;
      const int g0 = SG > 1 ? k0 * SG : group_of(a, k0);
      int c = k0 + w * per;
      const int end = min(k0 + kn, c + per);
      SB sb;
      sb.load(a, first, n0, g0, tid);
      Step<NB, RX> st[D];
#pragma unroll
      for (int d = 0; d < D; ++d) load(st[d], c + d);
      if (k0 > 0) __syncthreads();  // the block before is used up
      sb.store(a, sl, g0, tid);
      __syncthreads();
      auto mul = [&](Step<NB, RX>& b, int c) {
        const int at = SG > 1 ? (c - k0) * SG : group_of(a, c) - g0;
        multiply<DT, NB, SG, RX, ZERO, SB>(acc, b, bits, xl, sl, at, lane);
      };
      for (int left = (per + D - 1) / D; left > 1; --left, c += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
          if (c + d < end) mul(st[d], c + d);
          load(st[d], c + D + d);
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (c + d < end) mul(st[d], c + d);
    }
  }
}

// (Scheduled for four waves a SIMD, which is what a grid has of it: 64 experts 2048 x 2048 of 64 rows
// 27.3 -> 25.2 us, 16 x 4096 x 11007 12.8 -> 12.3. 32 columns with groups of 32 or 64 need the registers of two, or
// they go to scratch.)
template <int DT, int NB, int SG, int RX, bool ZERO, int W, int D>
__attribute__((amdgpu_waves_per_eu(NB > 1 && SG > 1 ? 2 : 4, 4)))
__global__ void __launch_bounds__(64 * W) gemm_int4_few(Args a) {
  constexpr int KB = 64;  // chunks whose scales are in LDS
  using SB = ScaleBlock<DT, 16 * NB, SG, KB, ZERO, 64 * W>;
  constexpr int XL = 4096, XS = W * (NB > 4 ? NB * 1024 : XL);  // a wave's rows of a chunk; later its sums
  static_assert(NB <= 4, "the sums reuse the rows' LDS");
  __shared__ __attribute__((aligned(1024))) char smem[XS + SB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  RowTile r;
  int tn;
  if (a.ends) {
    if (!find_tile<16>(a, blockIdx.x, lane, r, tn)) return;
  } else {
    tn = blockIdx.x % a.tiles_n;
    r.e = 0;
    r.row0 = blockIdx.x / a.tiles_n * 16;
    r.rows = min(16, a.T - r.row0);
    if (r.rows <= 0) return;
  }
  const int n0 = tn * (16 * NB);
  char* xl = smem + w * XL;
  char* sl = smem + XS;
  f32x4 acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  few_sums<DT, NB, SG, RX, ZERO, W, D, SB>(a, r, n0, tid, w, xl, sl, acc);

  float* red = (float*)smem;  // [wave][16 NB columns x 16 rows]
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[w * (NB * 256) + (j * 4 + v) * 64 + lane] = acc[j][v];
  __syncthreads();
  for (int at = tid; at < NB * 256; at += 64 * W) {
    const int ln = at & 63, v = (at >> 6) & 3, j = at >> 8;
    const int m = 4 * (ln >> 4) + v, n = n0 + j * 16 + (ln & 15);
    if (m >= r.rows || n >= a.N) continue;
    float s = red[at];
#pragma unroll
    for (int u = 1; u < W; ++u) s += red[u * (NB * 256) + at];
    ((unsigned short*)a.C)[((long long)r.row0 + m) * a.ldc + n] = (unsigned short)pack2<DT>(s, 0.f);
  }
}

// ---- more rows -----------------------------------------------------------
// A workgroup takes 16 MB rows x 64 NB columns: 4 column waves of 16 NB columns for
// each of KW parts of k (every KW-th chunk). The rows of KW chunks are staged through LDS, permuted on the way in ([row][256 B], 16-B piece c
// at c ^ (row & 15): conflict-free both ways), the next ones in registers
// meanwhile.
template <int DT, int MB, int NB, int SG, bool ZERO, int KW>
__global__ void __launch_bounds__(256 * KW) gemm_int4_rows(Args a) {
  constexpr int BM = 16 * MB, BN = 64 * NB, XB = BM * 256;  // bytes of a chunk's rows
  constexpr int THREADS = 256 * KW;
  constexpr int CH = XB / 16 / 256;                         // 16-B pieces a thread stages
  constexpr int XS = 2 * KW * XB;
  static_assert((KW - 1) * 4 * 64 * MB * NB * 16 <= XS, "the sums reuse the rows' LDS");
  constexpr int KB = 32;  // chunks whose scales are in LDS
  using SB = ScaleBlock<DT, BN, SG, KB, ZERO, THREADS>;
  static_assert(CH * 256 * 16 == XB, "whole pieces");
  __shared__ __attribute__((aligned(1024))) char smem[XS + SB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wc = w & 3, half = w >> 2;
  const int l16 = lane & 15, g = lane >> 4;

  RowTile r;
  int tn;
  if (a.ends) {
    if (!find_tile<BM>(a, blockIdx.x, lane, r, tn)) return;
  } else {
    // row tiles of one column tile side by side: the weight is read from memory once
    const int tm = (a.T + BM - 1) / BM;
    tn = blockIdx.x / tm;
    if (tn >= a.tiles_n) return;
    r.e = 0;
    r.row0 = blockIdx.x % tm * BM;
    r.rows = min(BM, a.T - r.row0);
  }
  const int n0 = tn * BN + wc * (16 * NB);
  const int K = r.e == a.E ? 0 : a.K;  // rows behind the last group: zeros
  const long long first = (long long)(r.e == a.E ? 0 : r.e) * a.N;
  const Weights<NB> weights(a, first, n0, lane);
  char* sl = smem + XS;
  const __amdgpu_buffer_rsrc_t xr = rows_buffer(a, r);

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nc = (K + 127) / 128, np = (nc + KW - 1) / KW;  // chunks, and steps of KW
  const Bits bits = Bits::make<DT>();
  u32x4 xs[CH], qn[NB], q[NB];
  int xo[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int at = tid + i * THREADS, row = at / (16 * KW);
    xo[i] = row < r.rows ? (row * (int)a.lda + at % (16 * KW) * 8) * 2 : kOutside;
  }
  // Rows and weights of a step (rows past K are zeros, weights repeat the last chunk)
  auto load = [&](int step) {
    weights.load(qn, KW * step + half, nc);
    const int left = K - step * (128 * KW);
#pragma unroll
    for (int i = 0; i < CH; ++i)
      xs[i] = load_row(xr, tid % (16 * KW) * 8 < left ? xo[i] : kOutside, left > 0 ? step * (256 * KW) : 0);
  };
  // Rows to LDS, weights to the operand's lanes: what the next step will use
  auto ready = [&](int step) {
    char* buf = smem + (step & 1) * KW * XB;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      q[j] = qn[j];
      to_operand(q[j], (l16 * 4 + g) * 4);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = tid + i * THREADS, row = at / (16 * KW), c = at % (16 * KW);
      *(lds_u32x4_t*)(buf + (c >> 4) * XB + row * 256 + (((c & 15) ^ (row & 15)) << 4)) =
          __builtin_bit_cast(u32x4, permute_row(xs[i]));
    }
  };
  SB sb;
  if (np > 0) {
    sb.load(a, first, tn * BN, 0, tid);
    load(0);
    ready(0);
    load(1);
  }
  int g0 = 0;
  for (int step = 0; step < np; ++step) {
    if (step % (KB / KW) == 0) {  // the scales of the next KB chunks
      g0 = SG > 1 ? KW * step * SG : group_of(a, KW * step);
      if (step) {
        sb.load(a, first, tn * BN, g0, tid);
        __syncthreads();  // those before are used up
      }
      sb.store(a, sl, g0, tid);
    }
    // this step's rows are written, and the other buffer's readers are done (loads stay in flight)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const char* xb = smem + (step & 1) * KW * XB + half * XB;
    u32x4 qc[NB];
    Scales<SG, DT, ZERO> s[NB];
    const int c = min(KW * step + half, nc - 1), at = SG > 1 ? c * SG - g0 : group_of(a, c) - g0;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      SB::read(s[j], sl, wc * (16 * NB) + 16 * j + l16, at);
      qc[j] = q[j];
    }
    // the next step's rows and operands, beside this one's products
    ready(step + 1);
    load(step + 2);
    constexpr int PER = 4 / SG;
    f32x4 p[MB][NB];
    Minus minus[NB];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s16x8 xf[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i)
        xf[i] = *(const lds_s16x8*)(xb + (16 * i + l16) * 256 + (((4 * t + g) ^ l16) << 4));
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (t % PER == 0) minus[j] = minus_of<DT>(s[j].zero(t / PER));
        const s16x8 wf = widen<DT>(qc[j][t], bits, minus[j]);
        const s16x8 mf = __builtin_bit_cast(s16x8, u32x4{minus[j].m[0], minus[j].m[1], minus[j].m[1], minus[j].m[1]});
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if (t % PER == 0) p[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
          p[i][j] = mfma16x16x32<DT>(xf[i], wf, p[i][j]);
        }
        if constexpr (DT == kBF16) {
#pragma unroll
          for (int i = 0; i < MB; ++i) p[i][j] = mfma16x16x32<DT>(xf[i], mf, p[i][j]);
        }
        if (t % PER == PER - 1) {
          const float sc = s[j].scale(t / PER);
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(sc, p[i][j][v], acc[i][j][v]);
        }
      }
    }
  }

  // the other K parts' sums to the first one's waves, added in order
  __syncthreads();
  float* red = (float*)smem + wc * (MB * NB * 256) + lane;
  if (half > 0) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          red[(half - 1) * (MB * NB * 1024) + ((i * NB + j) * 4 + v) * 64] = acc[i][j][v];
  }
  __syncthreads();
  if (half == 0) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float sum = acc[i][j][v];
#pragma unroll
          for (int u = 0; u < KW - 1; ++u) sum += red[u * (MB * NB * 1024) + ((i * NB + j) * 4 + v) * 64];
          const int m = 16 * i + 4 * g + v, n = n0 + 16 * j + l16;
          if (m < r.rows && n < a.N)
            ((unsigned short*)a.C)[((long long)r.row0 + m) * a.ldc + n] = (unsigned short)pack2<DT>(sum, 0.f);
        }
  }
}

// Row tiles x column tiles of a launch, as its kernel numbers them.
inline long long blocks_of(const Args& a, int bm, int bn) {
  const long long rows = a.ends ? row_tiles_bound(a.T, a.E, bm, a.zero_tail) : (a.T + bm - 1) / bm;
  return rows * ((a.N + bn - 1) / bn);
}

template <int DT, int NB, int SG, int RX, bool ZERO, int W>
hipError_t launch_few(Args a, hipStream_t s) {
  a.tiles_n = (a.N + 16 * NB - 1) / (16 * NB);
  const long long blocks = blocks_of(a, 16, 16 * NB);
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_int4_few<DT, NB, SG, RX, ZERO, W, 2>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(64 * W),
                     0, s, a);
  return hipGetLastError();
}

template <int DT, int MB, int NB, int SG, bool ZERO, int KW>
hipError_t launch_rows(Args a, hipStream_t s) {
  a.tiles_n = (a.N + 64 * NB - 1) / (64 * NB);
  const long long blocks = blocks_of(a, 16 * MB, 64 * NB);
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_int4_rows<DT, MB, NB, SG, ZERO, KW>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(256 * KW), 0, s,
                     a);
  return hipGetLastError();
}

// Row tiles of bm rows, as many as the rows fill on average where groups share them.
inline long long tiles_about(const Args& a, int bm) {
  if (!a.ends) return (a.T + bm - 1) / bm;
  const long long full = (a.T + (long long)a.E * bm / 2) / bm, groups = a.T < a.E ? a.T : a.E;
  return full > groups ? full : groups;
}

template <int DT, int SG, int RX, bool ZERO>
hipError_t pick_few(const Args& a, hipStream_t s) {
  // Waves a tile: enough to fill the CUs where there are few tiles (1 x 4096 x 4096: 8
  // waves 4.5 us, 4 5.2), no more where there are many — the chip starts about 3.5
  // waves a ns (16 x 4096 x 11007: 4 waves 11.7 us, 2 15.0; 64 experts 2048 x 2048 of
  // 64 rows, 32 columns a tile: 2 waves 27 us, 4 29, 8 43; 16 columns and 2 waves 30).
  const long long tiles = tiles_about(a, 16) * ((a.N + 15) / 16);
  // Long sums of many tiles: 8 waves on 32 columns (1 x 8192 x 16384: 14.9 us, 4 on 16 15.6;
  // 8 rows 18.5, 20; 64 rows of 16 experts 8192 x 2048 37, 42; but 77 of 8, 4128 x 1416: 14.8, 13.1).
  if (tiles >= 4096) return launch_few<DT, 2, SG, RX, ZERO, 2>(a, s);
  if (tiles > 512 && a.K >= 48 * 128) return launch_few<DT, 2, SG, RX, ZERO, 8>(a, s);
  if (tiles > 512) return launch_few<DT, 1, SG, RX, ZERO, 4>(a, s);
  return launch_few<DT, 1, SG, RX, ZERO, 8>(a, s);
}

template <int DT, int SG, bool ZERO>
hipError_t pick(const Args& a, hipStream_t s) {
  if (a.T <= 4) return pick_few<DT, SG, 1, ZERO>(a, s);
  if ((a.T + a.E - 1) / a.E <= 16) return pick_few<DT, SG, 4, ZERO>(a, s);
  // More rows than 16: the least of the times of the grids, in us. The tall tiles read
  // and widen the weights fewer times, but a workgroup of theirs fills a CU: a round of
  // 256 costs what one does (us a step of 512 k: 16 rows 1.0, 32 1.35, 64 1.95; of 64
  // rows x 128 columns a step of 256 k: 1.9). Tiles of 16 x 16 cost a step's latency a
  // wave, or the sum of their work. Measured, us: 25 x 1024 x 5632: 16 x 16 6.4, 32
  // rows 14.5; 33 x 448 x 5216 7.0, 32 rows 17, 64 23; 47 x 4480 x 10176 29, 27, 35;
  // 64 x 8192 x 4096 22, 15.5, 20; 64 x 16384 x 4096 35, 27, 21.5; 512 x 4096 x 4096: 64
  // rows 41, with 128 columns 35.
  const int chunks = (a.K + 127) / 128, steps = (chunks + 3) / 4;
  auto rounds = [&](int bm, int bn) { return (int)((tiles_about(a, bm) * ((a.N + bn - 1) / bn) + 255) / 256); };
  const double type = DT == kF16 ? 0.8 : 1.0;
  const double work = tiles_about(a, 16) * ((a.N + 15) / 16) * (double)chunks;
  const double few = work * 0.00035 > chunks * 0.08 ? work * 0.00035 : chunks * 0.08;
  const double t16 = 0.5 + type * 1.0 * rounds(16, 64) * steps, t32 = 0.5 + type * 1.35 * rounds(32, 64) * steps,
               t64 = 0.5 + type * 1.95 * rounds(64, 64) * steps,
               wide = 0.5 + type * 1.9 * rounds(64, 128) * ((chunks + 1) / 2);
  const double lo = t16 < t32 ? t16 : t32, hi = t64 < wide ? t64 : wide;
  if (few <= lo && few <= hi) return pick_few<DT, SG, 4, ZERO>(a, s);
  if (lo <= hi)
    return t16 < t32 ? launch_rows<DT, 1, 1, SG, ZERO, 4>(a, s) : launch_rows<DT, 2, 1, SG, ZERO, 4>(a, s);
  return t64 <= wide ? launch_rows<DT, 4, 1, SG, ZERO, 4>(a, s) : launch_rows<DT, 4, 2, SG, ZERO, 2>(a, s);
}

template <int DT, bool ZERO>
hipError_t pick_groups(const Args& a, int G, hipStream_t s) {
  return G == 32 ? pick<DT, 4, ZERO>(a, s) : G == 64 ? pick<DT, 2, ZERO>(a, s) : pick<DT, 1, ZERO>(a, s);
}

template <int DT>
hipError_t pick_zero(const Args& a, int G, hipStream_t s) {
  return a.zero ? pick_groups<DT, true>(a, G, s) : pick_groups<DT, false>(a, G, s);
}

}  // namespace kint4

hipError_t int4_gemm(const Int4Problem& p, hipStream_t stream) {
  if (p.N == 0 || p.T == 0 || p.E == 0) return hipSuccess;
  // a chunk's scales are whole groups: G divides 128 or is a multiple of it
  if (p.G < 32 || p.G % 32 || (p.G != 32 && p.G != 64 && p.G % 128) || p.K % p.G) return hipErrorInvalidValue;
  // row loads are 16 B, at offsets below 2^31 in a tile
  if ((uintptr_t)p.X % 16 || p.ldx % 8 || p.ldx > (1ll << 23) || p.K > (1 << 23)) return hipErrorInvalidValue;
  kint4::Args a{};
  a.A = p.X;
  a.B = p.q;
  a.C = p.C;
  a.ends = p.ends;
  a.ends64 = p.ends64;
  a.E = p.E;
  a.T = p.T;
  a.N = p.N;
  a.K = p.K;
  a.lda = p.ldx;
  a.ldc = p.ldc;
  a.zero_tail = p.zero_tail;
  a.scale = p.scale;
  a.zero = (const unsigned char*)p.zero;
  a.groups = p.K / p.G;
  a.scales = (long long)p.E * p.N * a.groups;
  a.chunk_g = p.G > 128 ? (unsigned)(((1ll << 32) + p.G / 128 - 1) / (p.G / 128)) : 0u;
  if (p.dtype == kBF16) return kint4::pick_zero<kBF16>(a, p.G, stream);
  if (p.dtype == kF16) return kint4::pick_zero<kF16>(a, p.G, stream);
  return hipErrorInvalidValue;
}

}  // namespace pdmb
