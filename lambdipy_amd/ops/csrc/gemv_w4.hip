// A few rows of activations times MX fp4 weights.
//
//   y[m, n] = sum_k x[m, k] * e2m1(w[n, k]) * 2^(sw[n, k/32] - 127)
//
// x in bf16 or fp16, or MX e4m3 with scales of its own. What has to move is
// the weights (0.53 B an element), so they go from memory straight into the
// registers of the one wave that multiplies them. The products are taken by
// the 16-bit MFMA with f32 sums: e2m1 and e4m3 values times their power of
// two are exact in bf16, and so is every product in f32. (The scaled
// f8f6f4 MFMA would take the bytes as they are, but does not hold its inner
// sums to f32: 2.7e-5 off over K = 512.)
//
// A wave takes 128 k a step of 16 weight rows a tile: lane (c, g) =
// (lane & 15, lane >> 4) loads the 16 B of row c's block g. The waves of a
// workgroup split K step by step, so that together they read neighbouring
// bytes of a row, and join their sums in LDS in a fixed order.

#include "lpx_common.h"
#include "kernels.h"

namespace lpx {

namespace {

typedef __bf16 nbf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 nbf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 nf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 nf16x8 __attribute__((ext_vector_type(8)));

enum { X_BF16, X_F16, X_MX };

struct W4Args {
  const unsigned char* x;   // bytes of bf16, fp16 or e4m3 rows
  const unsigned char* sx;  // MX only: [ceil(K/128)][M][4]
  const unsigned char* w;   // [N][K/2]
  const unsigned char* sw;  // [ceil(K/128)][N][4]
  void* y;                  // [M][N]
  long x_stride;            // bytes
  int M, N, K;
  bool bf16_out;
};

__device__ __forceinline__ i32x4 load16(const unsigned char* p) {
  i32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

__device__ __forceinline__ unsigned load4(const unsigned char* p) {
  unsigned v;
  __builtin_memcpy(&v, p, 4);
  return v;
}

// Byte i of a scale word as 2^(byte - 127); 2^-127 is an f32 subnormal.
__device__ __forceinline__ float scale_of(unsigned word, int i) {
  return __uint_as_float(max(((word >> (8 * i)) & 255u) << 23, 0x400000u));
}

// 8 e2m1 (one word) times s -> bf16
__device__ __forceinline__ nbf16x8 w_bf16(unsigned v, float s) {
  const nbf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 0);
  const nbf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 1);
  const nbf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 2);
  const nbf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 3);
  return nbf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ nf16x8 w_f16(unsigned v) {
  const nf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 0);
  const nf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 1);
  const nf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 2);
  const nf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 3);
  return nf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 e4m3 (two words) times s -> bf16
__device__ __forceinline__ nbf16x8 x_bf16(int lo, int hi, float s) {
  const nbf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  const nbf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const nbf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  const nbf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return nbf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Words r[0..3] of lane groups 0..3 transposed: word j of the result is, in
// group g, word g of group j.
__device__ __forceinline__ i32x4 transpose_groups(i32x4 r) {
  const auto a = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return i32x4{(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
}

// What one step of a wave multiplies.
template <int MODE, int MT, int NT>
struct Step {
  static constexpr int XW = MODE == X_MX ? 2 : 4;  // 16-B loads a row
  i32x4 w[NT];
  unsigned sw[NT];
  i32x4 x[MT][XW];
  unsigned sx[MT];
};

// MT x NT tiles of 16 rows of x by 16 rows of weights.
template <int MODE, int MT, int NT, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void gemv_w4_kernel(W4Args a) {
  typedef Step<MODE, MT, NT> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * NT * 16, m0 = (int)blockIdx.y * MT * 16;
  const int steps = (a.K + 127) >> 7;
  const bool half_last = (a.K & 127) != 0;

  // Rows behind the last are the last again; their sums are not stored.
  const unsigned char* wp[NT];
  const unsigned char* swp[NT];
  const unsigned char* xp[MT];
  const unsigned char* sxp[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min(n0 + t * 16 + c, a.N - 1);
    wp[t] = a.w + (long)n * (a.K >> 1) + g * 16;
    swp[t] = a.sw + (long)n * 4;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = min(m0 + t * 16 + c, a.M - 1);
    xp[t] = a.x + m * a.x_stride +
            (MODE == X_BF16 ? g * 64 : MODE == X_F16 ? g * 16
                                                     : (g >> 1) * 64 + (g & 1) * 16);
    sxp[t] = MODE == X_MX ? a.sx + (long)m * 4 : nullptr;
  }

  auto load = [&](S& f, int s) {
    // K may end after the first two blocks of the last step
    const bool half = half_last && s == steps - 1;
    const bool in = !half || g < 2;
    const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f.w[t] = in ? load16(wp[t] + (long)s * 64) : zero;
      f.sw[t] = load4(swp[t] + (long)s * a.N * 4);
      if (half) f.sw[t] &= 0xffffu;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if constexpr (MODE == X_MX) {
        f.x[t][0] = in ? load16(xp[t] + (long)s * 128) : zero;
        f.x[t][1] = in ? load16(xp[t] + (long)s * 128 + 32) : zero;
        f.sx[t] = load4(sxp[t] + (long)s * a.M * 4);
        if (half) f.sx[t] &= 0xffffu;
      } else if constexpr (MODE == X_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f.x[t][j] = in ? load16(xp[t] + (long)s * 256 + j * 16) : zero;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f.x[t][j] = !half || j < 2 ? load16(xp[t] + (long)s * 256 + j * 64)
                                     : zero;
      }
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};

  auto multiply = [&](const S& f) {
    if constexpr (MODE == X_F16) {
      // fp16 cannot hold every power of two, so here each MFMA takes one
      // block (its words spread over the lane groups) and the block's scale
      // goes onto the sum.
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const i32x4 w = transpose_groups(f.w[t]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const nf16x8 b = w_f16(w[j]);
          const float s = scale_of(f.sw[t], j);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                __builtin_bit_cast(nf16x8, f.x[i][j]), b, f32x4{0, 0, 0, 0}, 0,
                0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i][t][r] = __builtin_fmaf(p[r], s, acc[i][t][r]);
          }
        }
      }
    } else {
      // MFMA j takes elements [8j, 8j+8) of the four groups' blocks
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        nbf16x8 x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if constexpr (MODE == X_BF16)
            x[i] = __builtin_bit_cast(nbf16x8, f.x[i][j]);
          else
            x[i] = x_bf16(f.x[i][j >> 1][(j & 1) * 2],
                          f.x[i][j >> 1][(j & 1) * 2 + 1], scale_of(f.sx[i], g));
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const nbf16x8 b = w_bf16(f.w[t][j], scale_of(f.sw[t], g));
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                x[i], b, acc[i][t], 0, 0, 0);
        }
      }
    }
  };

  S f[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < steps) load(f[d], wave + d * WAVES);
  for (int s = wave; s < steps; s += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int now = s + d * WAVES;
      if (now < steps) {
        multiply(f[d]);
        if (now + DEPTH * WAVES < steps) load(f[d], now + DEPTH * WAVES);
      }
    }
  }

  // Join the waves' sums; then a thread owns four rows of one column.
  __shared__ f32x4 part[WAVES][MT * NT][64];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][i * NT + t][lane] = acc[i][t];
  __syncthreads();
  for (int e = (int)threadIdx.x; e < MT * NT * 64; e += WAVES * 64) {
    const int tile = e >> 6, l = e & 63;
    f32x4 v = part[0][tile][l];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += part[k][tile][l];
    const int n = n0 + (tile % NT) * 16 + (l & 15);
    const int m = m0 + (tile / NT) * 16 + (l >> 4) * 4;
    if (n >= a.N) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (m + r >= a.M) break;
      const long at = (long)(m + r) * a.N + n;
      if (a.bf16_out)
        static_cast<__bf16*>(a.y)[at] = (__bf16)v[r];
      else
        static_cast<float*>(a.y)[at] = v[r];
    }
  }
}

template <int MODE, int MT, int NT, int WAVES, int DEPTH>
hipError_t launch(const W4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + NT * 16 - 1) / (NT * 16)),
                  (unsigned)((a.M + MT * 16 - 1) / (MT * 16)));
  gemv_w4_kernel<MODE, MT, NT, WAVES, DEPTH>
      <<<grid, dim3(WAVES * 64), 0, stream>>>(a);
  return hipGetLastError();
}

template <int MODE>
hipError_t by_size(const W4Args& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  if (a.K < 64 || a.K % 64 != 0) return hipErrorInvalidValue;
  if (a.M <= 16) return launch<MODE, 1, 1, 8, 2>(a, stream);
  if (a.M <= 32) return launch<MODE, 2, 2, 8, 2>(a, stream);
  return launch<MODE, 4, 2, 4, 2>(a, stream);
}

}  // namespace

hipError_t gemv_w4(ActType t, const void* x, long x_stride,
                   const unsigned char* w, const unsigned char* sw, void* y,
                   bool bf16_out, int M, int N, int K, hipStream_t stream) {
  const W4Args a{static_cast<const unsigned char*>(x), nullptr, w, sw, y,
                 x_stride * 2, M, N, K, bf16_out};
  if (t == ActType::bf16) return by_size<X_BF16>(a, stream);
  if (t == ActType::f16) return by_size<X_F16>(a, stream);
  return hipErrorInvalidValue;
}

hipError_t gemv_mx_w4(const unsigned char* q, const unsigned char* sq,
                      const unsigned char* w, const unsigned char* sw, void* y,
                      bool bf16_out, int M, int N, int K, hipStream_t stream) {
  return by_size<X_MX>(W4Args{q, sq, w, sw, y, (long)K, M, N, K, bf16_out},
                       stream);
}

}  // namespace lpx
