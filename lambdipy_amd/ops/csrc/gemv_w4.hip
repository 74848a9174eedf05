// A few rows of activations times MX fp4 weights.
//
//   y[m, n] = sum_k x[m, k] * e2m1(w[n, k]) * 2^(sw[n, k/32] - 127)
//
// x in bf16 or fp16, or MX e4m3 with scales of its own. What has to move is
// the weights (0.53 B an element). The products are taken by the 16-bit MFMA
// with f32 sums: e2m1 and e4m3 values times their power of two are exact in
// bf16 (scale bytes of weights up to 252, of activations 3 to 246: more is
// infinite, less loses what is under 2^-133; 255 is NaN), and so is every
// product in f32. (The scaled f8f6f4 MFMA would take
// the bytes as they are, but does not hold its inner sums to f32: 2.7e-5 off
// over K = 512.)
//
// A wave takes 128 k a step: 16 rows of weights a tile, 16 rows of x a tile.
// The MFMA wants neighbouring lanes in different rows, the load path
// neighbouring lanes in one row (16 clocks a load of 1 KB then, 64
// otherwise, which bound everything but the smallest x), so each wave turns
// its steps round through LDS of its own, without a barrier. The waves of a
// workgroup split K step by step, so that together they read neighbouring
// bytes of a row, and join their sums in LDS in a fixed order.
//
// Measured: 100000 x 8192 by one bf16 row 74 us, 5.9 TB/s (reading alone
// reaches 6.4); 8192 x 8192 by 16 MX rows 8.1 us (10.6 where all of it comes
// from memory); 28000 x 8192 by 64 MX rows 38 and 45 us, of which the MFMA is
// busy 12 and the conversions to bf16, LDS and the load path about as long
// each; 437 tiles on 256 CUs leave a seventh of them idle. By 64 bf16 rows 45
// and 53, fp16 66 and 73.

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

// Of a scale that goes onto a sum: 255 is NaN. (The conversions take the
// infinity of scale_of as that.)
__device__ __forceinline__ float nan_or_scale_of(unsigned word, int i) {
  return ((word >> (8 * i)) & 255u) == 255u ? __builtin_nanf("") : scale_of(word, i);
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

// What a wave loads for one step, in the order of memory: neighbouring lanes
// hold neighbouring 16-B pieces of a row.
// FEW: of x only the rows that one load holds (4, of MX 8) are there.
template <int MODE, int MT, int NT, bool FEW>
struct Step {
  static constexpr int XL = FEW ? 1 : MODE == X_MX ? 2 : 4;  // loads a tile of x
  i32x4 w[NT];
  i32x4 x[MT][XL];
  unsigned sw, sx;  // of column, row `lane`
};

// Where a wave brings a step into the MFMA's order. The pieces of a row are
// permuted by the row, so that both the writes (along rows) and the reads
// (down 16 rows) meet every bank once.
template <int MODE, int MT, int NT, bool FEW>
struct Exchange {
  static constexpr int XTILE = Step<MODE, MT, NT, FEW>::XL * 1024;
  static_assert(NT <= 4 && MT <= 4, "a lane brings one scale of each side");
  // In LDS the scales cost less than between lanes, but 64 rows of 16 bits
  // leave no room for them where two workgroups are to share a CU's 160 KB.
  static constexpr bool SCALES = MODE == X_MX || MT < 4;
  unsigned char w[NT][1024];
  unsigned char x[MT][XTILE];
  unsigned sw[SCALES ? NT * 16 : 0], sx[MODE == X_MX ? MT * 16 : 0];
};

// MT x NT tiles of 16 rows of x by 16 rows of weights.
template <int MODE, int MT, int NT, int WAVES, int DEPTH, bool FEW>
__global__ __launch_bounds__(WAVES * 64) void gemv_w4_kernel(W4Args a) {
  static_assert(!FEW || MT == 1, "few rows are one tile");
  typedef Step<MODE, MT, NT, FEW> S;
  typedef Exchange<MODE, MT, NT, FEW> E;
  __shared__ union Shared {
    E exchange[WAVES];
    f32x4 part[WAVES][MT * NT][64];
    __device__ Shared() {}
  } sh;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int xc = FEW ? c & (MODE == X_MX ? 7 : 3) : c;
  // neighbouring tiles on one XCD: their scales share lines of its L2
  const int n0 = (int)lpx_xcd_swizzle(blockIdx.x, gridDim.x) * NT * 16;
  const int m0 = (int)blockIdx.y * MT * 16;
  const int steps = (a.K + 127) >> 7;
  const bool half_last = (a.K & 127) != 0;
  E& ex = sh.exchange[wave];

  // Rows behind the last are the last again; their sums are not stored.
  constexpr int WROW = 4;                        // pieces of a row a step
  constexpr int XROW = MODE == X_MX ? 8 : 16;
  const unsigned char* const w0 = a.w + (long)n0 * (a.K >> 1);
  const unsigned char* const x0 = a.x + m0 * a.x_stride;
  unsigned woff[NT], xoff[MT][S::XL];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    woff[t] = (unsigned)min(t * 16 + lane / WROW, a.N - 1 - n0) * (unsigned)(a.K >> 1) +
              lane % WROW * 16;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int l = 0; l < S::XL; ++l)
      xoff[i][l] = (unsigned)min(i * 16 + l * (64 / XROW) + lane / XROW, a.M - 1 - m0) *
                       (unsigned)a.x_stride + lane % XROW * 16;
  const unsigned swoff = (unsigned)min(lane % (NT * 16), a.N - 1 - n0) * 4;
  const unsigned sxoff = (unsigned)min(lane % (MT * 16), a.M - 1 - m0) * 4;

  // Turn i of a wave is step wave + i * WAVES. Loads are issued without a
  // branch, so that the compiler's waits count them: turns behind the last
  // step read that one again, and where K ends in the middle of the last
  // step, the second half of the pieces reads the first half again.
  // `turn_round` clears what was read in place of nothing.
  const int turns = (steps + WAVES - 1) / WAVES;
  auto load = [&](S& f, int turn) {
    const int s = min(wave + turn * WAVES, steps - 1);
    const bool half = half_last && s == steps - 1;
    const unsigned wback = half && lane % WROW >= WROW / 2 ? WROW / 2 * 16 : 0;
    const unsigned xback = half && lane % XROW >= XROW / 2 ? XROW / 2 * 16 : 0;
    const unsigned char* const w = w0 + (long)s * (WROW * 16);
    const unsigned char* const x = x0 + (long)s * (XROW * 16);
#pragma unroll
    for (int t = 0; t < NT; ++t) f.w[t] = load16(w + (woff[t] - wback));
    f.sw = load4(a.sw + ((long)s * a.N + n0) * 4 + swoff);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int l = 0; l < S::XL; ++l) f.x[i][l] = load16(x + (xoff[i][l] - xback));
    if constexpr (MODE == X_MX)
      f.sx = load4(a.sx + ((long)s * a.M + m0) * 4 + sxoff);
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};

  auto put = [](unsigned char* p, i32x4 v) { *reinterpret_cast<i32x4*>(p) = v; };
  auto get = [](const unsigned char* p) { return *reinterpret_cast<const i32x4*>(p); };
  // A wave's LDS operations are carried out in order; this keeps the
  // compiler to it.
  auto in_order = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  auto wat = [](int row, int piece) { return (row * 4 + (piece ^ (row >> 2))) * 16; };
  auto xat = [](int row, int piece) {
    return MODE == X_MX ? (row * 8 + (piece ^ (row >> 1))) * 16
                        : (row * 16 + (piece ^ row)) * 16;
  };

  // What a lane multiplies: its block of each tile's rows, as loaded.
  struct Turned {
    i32x4 w[NT], x[MT][MODE == X_MX ? 2 : 4];
    unsigned sw[NT], sx[MT];
  };
  auto turn_round = [&](const S& f, Turned& q, int turn) {
    const int s = wave + turn * WAVES;
    const bool none = s >= steps;
    const bool part = none || (half_last && s == steps - 1);
    const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NT; ++t) put(ex.w[t] + wat(lane / WROW, lane % WROW), f.w[t]);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int l = 0; l < S::XL; ++l)
        put(ex.x[i] + xat(l * (64 / XROW) + lane / XROW, lane % XROW), f.x[i][l]);
    const unsigned sw = part ? f.sw & 0xffffu : f.sw;
    if constexpr (E::SCALES) ex.sw[lane % (NT * 16)] = sw;
    if constexpr (MODE == X_MX)
      ex.sx[lane % (MT * 16)] = part ? f.sx & 0xffffu : f.sx;
    in_order();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      q.w[t] = get(ex.w[t] + wat(c, g));
      if constexpr (E::SCALES)
        q.sw[t] = ex.sw[t * 16 + c];
      else
        q.sw[t] = (unsigned)__shfl((int)sw, t * 16 + c, 64);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (MODE == X_MX) {
        // a lane's block lies in the pieces of two quarters
        const int at = (g >> 1) * 4 + (g & 1);
        q.x[i][0] = get(ex.x[i] + xat(xc, at));
        q.x[i][1] = get(ex.x[i] + xat(xc, at + 2));
        q.sx[i] = ex.sx[i * 16 + c];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q.x[i][j] = get(ex.x[i] + xat(xc, MODE == X_F16 ? 4 * j + g : 4 * g + j));
      }
    }
    in_order();
    if (part) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (none || g >= 2) q.w[t] = zero;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < (MODE == X_MX ? 2 : 4); ++j)
          if (none || (MODE == X_F16 ? j >= 2 : g >= 2)) q.x[i][j] = zero;
    }
  };

  auto multiply = [&](Turned& q) {
    if constexpr (MODE == X_F16) {
#pragma unroll
      for (int t = 0; t < NT; ++t) q.w[t] = transpose_groups(q.w[t]);
    }
    // A quarter of the step at a time, so that the next quarter's conversions
    // go on beside this one's MFMAs.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      i32x4 b[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        b[t] = MODE == X_F16
                   ? __builtin_bit_cast(i32x4, w_f16(q.w[t][j]))
                   : __builtin_bit_cast(i32x4, w_bf16(q.w[t][j], scale_of(q.sw[t], g)));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        i32x4 x;
        if constexpr (MODE == X_MX) {
          const i32x4 v = q.x[i][j / 2];
          x = __builtin_bit_cast(
              i32x4, x_bf16(v[j % 2 * 2], v[j % 2 * 2 + 1], scale_of(q.sx[i], g)));
        } else {
          x = q.x[i][j];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (MODE == X_F16) {
            // fp16 cannot hold every power of two, so here each MFMA takes
            // one block (its words spread over the lane groups) and the
            // block's scale goes onto the sum
            const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                __builtin_bit_cast(nf16x8, x), __builtin_bit_cast(nf16x8, b[t]),
                f32x4{0, 0, 0, 0}, 0, 0, 0);
            const float sc = nan_or_scale_of(q.sw[t], j);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i][t][r] = __builtin_fmaf(p[r], sc, acc[i][t][r]);
          } else {
            // MFMA j takes elements [8j, 8j+8) of the four groups' blocks
            acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(nbf16x8, x), __builtin_bit_cast(nbf16x8, b[t]),
                acc[i][t], 0, 0, 0);
          }
        }
      }
    }
  };

  // The next step's loads stay in front of a step's products (0x78f: all but
  // vector memory's instructions may pass); left to itself the compiler puts
  // them behind, which saves registers.
  constexpr int MAY_PASS = 0x78f;

  S f[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(f[d], d);
  int turn = 0;
  for (; turn + DEPTH < turns; turn += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Turned q;
      turn_round(f[d], q, turn + d);
      load(f[d], turn + d + DEPTH);  // on its way while this one is multiplied
      __builtin_amdgcn_sched_barrier(MAY_PASS);
      multiply(q);
    }
  }
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (turn + d < turns) {
      Turned q;
      turn_round(f[d], q, turn + d);
      multiply(q);
    }

  // Join the waves' sums; then a thread owns four rows of one column.
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sh.part[wave][i * NT + t][lane] = acc[i][t];
  __syncthreads();
  for (int e = (int)threadIdx.x; e < MT * NT * 64; e += WAVES * 64) {
    const int tile = e >> 6, l = e & 63;
    f32x4 v = sh.part[0][tile][l];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += sh.part[k][tile][l];
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

template <int MODE, int MT, int NT, int WAVES, int DEPTH, bool FEW = false>
hipError_t launch(const W4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + NT * 16 - 1) / (NT * 16)),
                  (unsigned)((a.M + MT * 16 - 1) / (MT * 16)));
  gemv_w4_kernel<MODE, MT, NT, WAVES, DEPTH, FEW>
      <<<grid, dim3(WAVES * 64), 0, stream>>>(a);
  return hipGetLastError();
}

// The largest tile of which more than half of the CUs get one: a wave loads
// and converts x once for all the weight rows of its tile, so that wide tiles
// cost less a weight, but half as wide ones on twice the CUs take less time.
// Up to a tile a CU its waves split K eight ways; with more, four ways, and
// two tiles share a CU; where half of the CUs have none, sixteen ways. us, weights from memory, K = 8192 but where given:
//   64 MX rows: N = 8192 2x4 tiles 15.0, 2x2 18.0; 12000 4x4 22.7, 2x4 25.8;
//     28000 4x4 by four waves 43.8, by eight 44.6; 50000 (K = 4096) 42.9, 48.0
//   32: 8192 2x2 12.3, 1x4 12.9; 12000 2x4 16.8, 2x2 21.0
//   16: 8192 1x2 10.0, 1x4 13.3; 12000 1x4 14.5, 1x2 16.4
//     2000 1x1 by sixteen waves 6.0, by eight 6.4
//   64 bf16 rows: 28000 4x4 by four waves 52.8, by eight 56.1
//   1: 1000 by sixteen waves 4.3, by eight 4.5; fp16 4.8, 5.3
template <int MODE>
hipError_t by_size(const W4Args& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  if (a.K < 64 || a.K % 64 != 0 || a.K > (1 << 24)) return hipErrorInvalidValue;
  constexpr long CUS = 256;
  auto tiles = [&](int mt, int nt) {
    return (long)((a.M + 16 * mt - 1) / (16 * mt)) * ((a.N + 16 * nt - 1) / (16 * nt));
  };
  auto fills = [&](int mt, int nt) { return tiles(mt, nt) > CUS / 2; };
  // Rows that one load of x holds: 100000 x 8192 by one bf16 row 73 us,
  // loading a tile of 16 rows of x 80 us.
  if (a.M <= (MODE == X_MX ? 8 : 4))
    return fills(1, 2)   ? launch<MODE, 1, 2, 8, 2, true>(a, stream)
           : fills(1, 1) ? launch<MODE, 1, 1, 8, 2, true>(a, stream)
                         : launch<MODE, 1, 1, 16, 2, true>(a, stream);
  if constexpr (MODE != X_F16)  // whose scaled sums do not fit the registers
    if (a.M > 32 && fills(4, 4))
      return tiles(4, 4) > CUS ? launch<MODE, 4, 4, 4, 1>(a, stream)
                               : launch<MODE, 4, 4, 8, 1>(a, stream);
  if (a.M > 16 && fills(2, 4)) {
    if constexpr (MODE != X_F16)  // 28000 x 8192 by 64: 72.9 us, by eight 66.8
      if (tiles(2, 4) > CUS) return launch<MODE, 2, 4, 4, 1>(a, stream);
    return launch<MODE, 2, 4, 8, 1>(a, stream);
  }
  if (a.M > 16 && fills(2, 2)) return launch<MODE, 2, 2, 8, 1>(a, stream);
  if (fills(1, 4)) return launch<MODE, 1, 4, 8, 1>(a, stream);
  if (fills(1, 2)) return launch<MODE, 1, 2, 8, 1>(a, stream);
  if (fills(1, 1)) return launch<MODE, 1, 1, 8, 1>(a, stream);
  return launch<MODE, 1, 1, 16, 2>(a, stream);
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
