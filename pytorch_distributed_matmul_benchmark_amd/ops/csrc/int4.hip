// int4.hip — products of a few rows with 4-bit weights and group scales:
//   C[r][n] = sum over groups j of scale[n][j] * sum over k in group j of X[r][k] (q[n][k] - zero[n][j])
// for bf16 / fp16 rows, one weight or (grouped by expert) one for each group
// of rows.
//
// Exactness: the nibbles go into the matrix instructions as whole numbers, so
// a weight is never rounded: bits of 16 + q are formed by one shift and one
// and-or for two values (16 .. 31 have the step 1 at a fixed mantissa place:
// bf16 0x4180 | q << 3, fp16 0x4c00 | q << 6). fp16 subtracts 16 + zero
// exactly (v_pk_add_f16); bf16, which has no packed add, adds a second product with the
// constant -(16 + zero), also a whole number, to the same fp32 sum. Each
// group's fp32 sum is scaled once, in fp32. (A row of X with an infinity
// gives NaN in bf16: the two products cancel.)
//
// A wave takes 16 NB columns and every W-th chunk of 128 k: lane (l16, g)
// loads 16 bytes (32 nibbles) of column l16 at byte 16 g of its 64-byte run.
// Four dwords a lane are transposed among the four 16-lane rows (two
// v_permlane32_swap, two v_permlane16_swap) so that the lane's dword j holds k
// 32 j + 8 g .. + 7: MFMA j then covers 32 consecutive k, the smallest group.
// A dword's halves hold nibbles i and i + 4; the row fragments are permuted
// the same way. The W waves' sums meet in LDS, added in wave order.
#include "api.h"
#include "grouped.h"

namespace pdmb {
namespace kint4 {

struct Args : GroupArgs {
  const void* scale;
  const unsigned char* zero;
  int groups;   // K / G
  int chunk_g;  // 128-k chunks of one group (G >= 128), else 1
};

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

// 8 nibbles as 16 + q (bf16) or q - zero (fp16; minus = -(16 + zero) twice)
template <int DT>
__device__ __forceinline__ s16x8 widen(unsigned d, unsigned minus) {
  u32x4 v;
  if constexpr (DT == kBF16) {
    v = u32x4{((d << 3) & 0x00780078u) | 0x41804180u, ((d >> 1) & 0x00780078u) | 0x41804180u,
              ((d >> 5) & 0x00780078u) | 0x41804180u, ((d >> 9) & 0x00780078u) | 0x41804180u};
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 m = __builtin_bit_cast(f16x2, minus);
    v = u32x4{((d << 6) & 0x03c003c0u) | 0x4c004c00u, ((d << 2) & 0x03c003c0u) | 0x4c004c00u,
              ((d >> 2) & 0x03c003c0u) | 0x4c004c00u, ((d >> 6) & 0x03c003c0u) | 0x4c004c00u};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, (unsigned)v[i]) + m);
  }
  return __builtin_bit_cast(s16x8, v);
}

// SG: scales of a 128-k chunk (G = 32: 4, 64: 2, 128 and more: 1).
template <int MB, int NB, int SG>
struct Stage {
  u32x4 q[NB], x[MB][4];
  unsigned short s[NB][SG];
  unsigned char z[NB][SG];
};

template <int DT, int MB, int NB, int SG, int W>
__global__ void __launch_bounds__(64 * W) gemm_int4(Args a) {
  __shared__ float red[W][MB * NB * 4 * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;

  RowTile r;
  int tn;
  if (a.ends) {
    if (!find_tile<16 * MB>(a, blockIdx.x, lane, r, tn)) return;
  } else {
    tn = blockIdx.x % a.tiles_n;
    r.e = 0;
    r.row0 = blockIdx.x / a.tiles_n * (16 * MB);
    r.rows = min(16 * MB, a.T - r.row0);
    if (r.rows <= 0) return;
  }
  const int n0 = tn * (16 * NB);
  const int K = r.e == a.E ? 0 : a.K;  // rows behind the last group: zeros
  const long long col = (long long)(r.e == a.E ? 0 : r.e) * a.N;

  const unsigned char* qp[NB];
  const unsigned short* sp[NB];
  const unsigned char* zp[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const long long n = col + min(n0 + 16 * j + l16, a.N - 1);
    qp[j] = (const unsigned char*)a.B + n * (a.K / 2) + 16 * g;
    sp[j] = (const unsigned short*)a.scale + n * a.groups;
    zp[j] = a.zero + n * a.groups;
  }
  const unsigned short* xp = (const unsigned short*)a.A + ((long long)r.row0 + l16) * a.lda + 8 * g;

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nc = (K + 127) / 128;
  auto load = [&](Stage<MB, NB, SG>& st, int c) {
    const int k0 = c * 128;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      st.q[j] = u32x4{0u, 0u, 0u, 0u};
      if (k0 + 32 * g < K) st.q[j] = __builtin_nontemporal_load((const u32x4*)(qp[j] + c * 64));
      const int s0 = SG > 1 ? c * SG : c / a.chunk_g;
#pragma unroll
      for (int t = 0; t < SG; ++t) {
        const int at = min(s0 + t, a.groups - 1);
        st.s[j][t] = sp[j][at];
        st.z[j][t] = a.zero ? zp[j][at] : 8;
      }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        st.x[i][t] = u32x4{0u, 0u, 0u, 0u};
        if (16 * i + l16 < r.rows && k0 + 32 * t + 8 * g < K)
          __builtin_memcpy(&st.x[i][t], xp + 16ll * i * a.lda + k0 + 32 * t, 16);
      }
  };
  Stage<MB, NB, SG> cur, nxt;
  int c = w;
  if (c < nc) load(cur, c);
  for (; c < nc; c += W) {
    if (c + W < nc) load(nxt, c + W);
    f32x4 p[MB][NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) transpose4(cur.q[j]);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      constexpr int PER = 4 / SG;  // MFMAs of a group
      s16x8 xf[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i) xf[i] = permute_row(cur.x[i][t]);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float off = 16.0f + (float)cur.z[j][t / PER];
        const unsigned minus = pack2<DT>(-off, -off);
        const s16x8 wf = widen<DT>(cur.q[j][t], minus);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if (t % PER == 0) p[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
          p[i][j] = mfma16x16x32<DT>(xf[i], wf, p[i][j]);
          if constexpr (DT == kBF16)
            p[i][j] = mfma16x16x32<DT>(xf[i], __builtin_bit_cast(s16x8, u32x4{minus, minus, minus, minus}), p[i][j]);
          if (t % PER == PER - 1) {
            const float s = to_f32<DT>(cur.s[j][t / PER]);
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(s, p[i][j][v], acc[i][j][v]);
          }
        }
      }
    }
    cur = nxt;
  }

  // the waves' sums, in wave order
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) red[w][((i * NB + j) * 4 + v) * 64 + lane] = acc[i][j][v];
  __syncthreads();
#pragma unroll
  for (int at = tid; at < MB * NB * 256; at += 64 * W) {
    float s = red[0][at];
#pragma unroll
    for (int v = 1; v < W; ++v) s += red[v][at];
    const int ln = at & 63, v = (at >> 6) & 3, ij = at >> 8;
    const int m = ij / NB * 16 + 4 * (ln >> 4) + v, n = n0 + ij % NB * 16 + (ln & 15);
    if (m < r.rows && n < a.N)
      ((unsigned short*)a.C)[((long long)r.row0 + m) * a.ldc + n] = (unsigned short)pack2<DT>(s, 0.f);
  }
}

template <int DT, int MB, int NB, int SG>
hipError_t launch(Args a, hipStream_t s) {
  constexpr int W = 8;
  a.tiles_n = (a.N + 16 * NB - 1) / (16 * NB);
  const long long rows = a.ends ? row_tiles_bound(a.T, a.E, 16 * MB, a.zero_tail) : (a.T + 16 * MB - 1) / (16 * MB);
  const long long blocks = rows * a.tiles_n;
  if (blocks > (1ll << 30)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_int4<DT, MB, NB, SG, W>), dim3((unsigned)((blocks + 7) / 8 * 8)), dim3(64 * W), 0, s, a);
  return hipGetLastError();
}

template <int DT, int SG>
hipError_t pick(const Args& a, hipStream_t s) {
  const int avg = (a.T + a.E - 1) / a.E;
  if (avg <= 16) return launch<DT, 1, 1, SG>(a, s);
  if (avg <= 32) return launch<DT, 2, 2, SG>(a, s);
  return launch<DT, 4, 2, SG>(a, s);
}

template <int DT>
hipError_t pick_groups(const Args& a, int G, hipStream_t s) {
  return G == 32 ? pick<DT, 4>(a, s) : G == 64 ? pick<DT, 2>(a, s) : pick<DT, 1>(a, s);
}

}  // namespace kint4

hipError_t int4_gemm(const Int4Problem& p, hipStream_t stream) {
  if (p.N == 0 || p.T == 0 || p.E == 0) return hipSuccess;
  // a chunk's scales are whole groups: G divides 128 or is a multiple of it
  if (p.G < 32 || p.G % 32 || (p.G != 32 && p.G != 64 && p.G % 128) || p.K % p.G) return hipErrorInvalidValue;
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
  a.chunk_g = p.G >= 128 ? p.G / 128 : 1;
  if (p.dtype == kBF16) return kint4::pick_groups<kBF16>(a, p.G, stream);
  if (p.dtype == kF16) return kint4::pick_groups<kF16>(a, p.G, stream);
  return hipErrorInvalidValue;
}

}  // namespace pdmb
