// Residual addition + root-mean-square norm, with the result in the input's
// type or as MX e4m3 (the layout that the MX GEMMs read).
//
//   h = x + r                        (f32; stored rounded once to x's type)
//   y = h * (mean(h^2) + eps)^-1/2 * w
//   MX: per 32 elements 2^e, the smallest power of two with
//       max|y| / 2^e <= 448; payload e4m3(y / 2^e), scale byte e + 127
//
// The norm is taken of the unrounded f32 sum, y is rounded once, and the sum
// of squares is held in f32 (a thread's terms in turn, then a tree).
//
// The row stays in registers between the two uses of it, so each input is
// read once and each output written once; memory bounds it. A thread owns 8
// neighbouring elements (16-B loads of 16-bit types), an MX block is four
// neighbouring lanes, a 128-element scale tile sixteen. A thread takes one
// step, or two, and a row as many threads as it needs: 16384 x 8192 bf16 with
// residual to MX 204 us with 256 threads of four steps each, 174 with 1024 of
// one, 162 where the stores also pass by the caches, 158 (6.0 TB/s) without
// the code for widths that are no multiple of 8; a copy of 2 GiB by a
// kernel of this form reaches 6.0, torch's 4.9.

#include <algorithm>

#include "lpx_common.h"
#include "kernels.h"

namespace lpx {

namespace {

typedef __bf16 nbf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 nf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef nbf16x8 type; };
template <> struct Vec8<_Float16> { typedef nf16x8 type; };
template <> struct Vec8<float> { typedef f32x8 type; };

// Rows of odd length start at any multiple of the element size; global
// memory takes wide accesses there.
template <typename T>
__device__ __forceinline__ f32x8 load8(const T* p) {
  typename Vec8<T>::type v;
  __builtin_memcpy(&v, p, sizeof(v));
  return __builtin_convertvector(v, f32x8);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, f32x8 f) {
  typedef int words __attribute__((ext_vector_type(sizeof(T) * 2), aligned(sizeof(T))));
  const typename Vec8<T>::type v =
      __builtin_convertvector(f, typename Vec8<T>::type);
  __builtin_nontemporal_store(__builtin_bit_cast(words, v),
                              reinterpret_cast<words*>(p));
}

// Elements [c, c+8) of a row of K; what lies behind K is 0. WHOLE: K is a
// multiple of 8.
template <bool WHOLE, typename T>
__device__ __forceinline__ f32x8 load_row(const T* row, int c, int K) {
  if (WHOLE || c + 8 <= K) return load8(row + c);
  if ((K & 7) == 1) return f32x8{(float)row[c], 0, 0, 0, 0, 0, 0, 0};
  // All are asked for before one is waited for, the last again in place of
  // those behind it: 9999 x 5004 fp16 104 us with a branch each, 96 so.
  T e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = row[min(c + j, K - 1)];
  f32x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < K ? (float)e[j] : 0.f;
  return v;
}

template <bool WHOLE, typename T>
__device__ __forceinline__ void store_row(T* row, int c, int K, f32x8 v) {
  if (WHOLE || c + 8 <= K) {
    store8(row + c, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c + j < K) row[c + j] = (T)v[j];
}

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[16];
  v = lpx_wave_allreduce_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
  for (unsigned i = 0; i < blockDim.x / 64; ++i) v += part[i];
  return v;
}

// E8M0 byte of a block: 448 = 1.75 * 2^8, so e = exponent - 8, one more where
// the significand is over 1.75. A block of zeros gets 2^0.
__device__ __forceinline__ unsigned mx_scale_byte(float amax) {
  const unsigned b = __float_as_uint(amax);
  if (b == 0) return 127u;
  const int s = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u);
  return s < 0 ? 0u : (unsigned)s;
}

// y[c .. c+8) as MX e4m3. All lanes of the wave come here together; lanes
// with c >= K bring zeros and store nothing. A row's lanes are neighbours, 8
// (K = 64) or a multiple of 16.
__device__ __forceinline__ void store_mx(unsigned char* __restrict__ qrow,
                                         unsigned char* __restrict__ sc,
                                         int row, int R, int c, int K,
                                         f32x8 y) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
  amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 2, 64));
  const unsigned byte = mx_scale_byte(amax);
  const float scale = __uint_as_float(byte << 23);
  unsigned tile = byte << (8 * ((c >> 5) & 3));
  tile |= __shfl_xor(tile, 4, 64);
  const unsigned more = __shfl_xor(tile, 8, 64);
  tile |= K > 64 ? more : 0x7f7f0000u;
  if (c >= K) return;
  i32x2 out;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    s16x2 t = {0, 0};
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, y[4 * u], y[4 * u + 1],
                                                 scale, false);
    t = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(t, y[4 * u + 2], y[4 * u + 3],
                                                 scale, true);
    out[u] = __builtin_bit_cast(int, t);
  }
  // 64-groups are kept as their quarters [q0 | q2 | q1 | q3]
  const int quarter = (c >> 4) & 3;
  const int slot = ((quarter & 1) << 1) | (quarter >> 1);
  __builtin_nontemporal_store(
      out, reinterpret_cast<i32x2*>(qrow + (c & ~63) + slot * 16 + (c & 8)));
  if ((c & 127) == 0)
    *reinterpret_cast<unsigned*>(sc + ((long)(c >> 7) * R + row) * 4) = tile;
}

struct NormArgs {
  const void* x;
  const void* res;     // may be null
  const void* weight;  // x's type, or f32
  void* h;             // written if res is given
  void* y;             // x's type, or the e4m3 payload
  unsigned char* sc;
  long x_stride, res_stride;  // elements
  int R, K;
  int first;  // row of the launch's first
  float eps;
  bool weight_f32;
};

template <typename T, bool MX, bool WHOLE>
__device__ __forceinline__ void finish8(const NormArgs& a, int row, int c,
                                        f32x8 h, float inv) {
  f32x8 w = {0, 0, 0, 0, 0, 0, 0, 0};
  if (c < a.K)
    w = a.weight_f32 ? load_row<WHOLE>((const float*)a.weight, c, a.K)
                     : load_row<WHOLE>((const T*)a.weight, c, a.K);
  const f32x8 y = h * inv * w;
  if constexpr (MX)
    store_mx((unsigned char*)a.y + (long)row * a.K, a.sc, row, a.R, c, a.K, y);
  else if (c < a.K)
    store_row<WHOLE>((T*)a.y + (long)row * a.K, c, a.K, y);
}

template <typename T, bool WHOLE>
__device__ __forceinline__ f32x8 read_h(const NormArgs& a, int row, int c,
                                        bool keep) {
  f32x8 h = load_row<WHOLE>((const T*)a.x + (long)row * a.x_stride, c, a.K);
  if (a.res) {
    h += load_row<WHOLE>((const T*)a.res + (long)row * a.res_stride, c, a.K);
    if (keep) store_row<WHOLE>((T*)a.h + (long)row * a.K, c, a.K, h);
  }
  return h;
}

__device__ __forceinline__ float square_sum(f32x8 h) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += h[j] * h[j];
  return s;
}

// Rows of at most 512: `lanes` (a power of two, 8 at least) of a wave each.
template <typename T, bool MX, bool WHOLE>
__global__ __launch_bounds__(256) void rmsnorm_short_kernel(NormArgs a, int lanes) {
  const int rows = 256 / lanes;
  const int row = a.first + (int)lpx_xcd_swizzle(blockIdx.x, gridDim.x) * rows +
                  (int)threadIdx.x / lanes;
  const int c = row < a.R ? (int)threadIdx.x % lanes * 8 : a.K;
  f32x8 h = {0, 0, 0, 0, 0, 0, 0, 0};
  if (c < a.K) h = read_h<T, WHOLE>(a, row, c, true);
  float s = square_sum(h);
  for (int m = lanes / 2; m > 0; m >>= 1) s += __shfl_xor(s, m, 64);
  finish8<T, MX, WHOLE>(a, row, c, h, rsqrtf(s / (float)a.K + a.eps));
}

// Rows of at most blockDim * STEPS * 8 elements.
template <typename T, bool MX, bool WHOLE, int STEPS>
__global__ __launch_bounds__(1024) void rmsnorm_kernel(NormArgs a) {
  // neighbouring rows on one XCD: their scale bytes share lines of its L2
  const int row = a.first + (int)lpx_xcd_swizzle(blockIdx.x, gridDim.x);
  f32x8 h[STEPS];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = (int)(i * blockDim.x + threadIdx.x) * 8;
    h[i] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (c < a.K) h[i] = read_h<T, WHOLE>(a, row, c, true);
    s += square_sum(h[i]);
  }
  const float inv = rsqrtf(block_sum(s) / (float)a.K + a.eps);
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    finish8<T, MX, WHOLE>(a, row, (int)(i * blockDim.x + threadIdx.x) * 8, h[i], inv);
}

// Longer rows: read a second time (the first pass left them in the caches).
template <typename T, bool MX, bool WHOLE>
__global__ __launch_bounds__(1024) void rmsnorm_long_kernel(NormArgs a) {
  const int row = a.first + (int)lpx_xcd_swizzle(blockIdx.x, gridDim.x);
  const int steps = (a.K + 8191) / 8192;
  float s = 0.f;
  for (int i = 0; i < steps; ++i) {
    const int c = (i * 1024 + (int)threadIdx.x) * 8;
    if (c < a.K) s += square_sum(read_h<T, WHOLE>(a, row, c, true));
  }
  const float inv = rsqrtf(block_sum(s) / (float)a.K + a.eps);
  for (int i = 0; i < steps; ++i) {
    const int c = (i * 1024 + (int)threadIdx.x) * 8;
    f32x8 h = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < a.K) h = read_h<T, WHOLE>(a, row, c, false);
    finish8<T, MX, WHOLE>(a, row, c, h, inv);
  }
}

// Whether rows of up to 1024 threads of one step are better done by half as
// many of two. Rows that the chip holds at once are not (512 x 5120 bf16 5.6
// us, 6.7 by two). Where that leaves a second round with little in it they
// are: 1030 x 4096 bf16 6.2 and 5.1, 2048 x 4096 14.2 and 16.1, 1000 x 7168
// 13.7 and 11.5, 8192 x 7168 84 and 88. So they are, however many, at 10 to 12
// waves, of which a CU takes two workgroups only (8192 x 5120 to MX 64 and 58;
// f32 63 and 67), and at widths off the loads' 8 (9999 x 5003 fp16 106 and 91).
template <typename T, bool WHOLE>
bool two_steps(int R, int waves) {
  const int slots = 256 * (waves > 9 ? 2 : 32 / waves);
  if (R <= slots) return false;
  if (sizeof(T) == 2 && (!WHOLE || (waves >= 10 && waves <= 12))) return true;
  return R <= (waves > 8 ? 2 * slots : slots + slots / 4);
}

// `each` rows to a workgroup of `threads`. A grid's threads are counted in 32
// bits, so that very many rows take more than one.
template <typename Kernel, typename... More>
hipError_t launch_rows(Kernel kernel, NormArgs a, int each, int threads,
                       hipStream_t stream, More... more) {
  const int most = 0x7fffffff / threads;  // workgroups
  for (long first = 0; first < a.R; first += (long)most * each) {
    const long left = (a.R - first + each - 1) / each;
    const dim3 grid((unsigned)std::min<long>(left, most)), block((unsigned)threads);
    a.first = (int)first;
    kernel<<<grid, block, 0, stream>>>(a, more...);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, bool MX, bool WHOLE>
hipError_t launch(const NormArgs& a, hipStream_t stream) {
  const int threads = (a.K + 7) / 8;
  if (threads <= 64) {
    int lanes = 8;
    while (lanes < threads) lanes *= 2;
    return launch_rows(rmsnorm_short_kernel<T, MX, WHOLE>, a, 256 / lanes, 256, stream, lanes);
  }
  const int waves = (threads + 63) / 64;
  if (threads <= 1024 && two_steps<T, WHOLE>(a.R, waves))
    return launch_rows(rmsnorm_kernel<T, MX, WHOLE, 2>, a, 1, (waves + 1) / 2 * 64, stream);
  if (threads <= 1024)
    return launch_rows(rmsnorm_kernel<T, MX, WHOLE, 1>, a, 1, waves * 64, stream);
  if (threads <= 2048)
    return launch_rows(rmsnorm_kernel<T, MX, WHOLE, 2>, a, 1, 1024, stream);
  return launch_rows(rmsnorm_long_kernel<T, MX, WHOLE>, a, 1, 1024, stream);
}

template <typename T, bool MX>
hipError_t by_width(const NormArgs& a, hipStream_t stream) {
  if constexpr (!MX)  // whose rows are whole blocks
    if (a.K % 8 != 0) return launch<T, MX, false>(a, stream);
  return launch<T, MX, true>(a, stream);
}

template <bool MX>
hipError_t by_type(ActType t, const NormArgs& a, hipStream_t stream) {
  if (a.R <= 0) return hipSuccess;
  if (a.K <= 0 || (MX && a.K % 64 != 0)) return hipErrorInvalidValue;
  switch (t) {
    case ActType::bf16: return by_width<__bf16, MX>(a, stream);
    case ActType::f16: return by_width<_Float16, MX>(a, stream);
    case ActType::f32: return by_width<float, MX>(a, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t rmsnorm(ActType t, const void* x, long x_stride, const void* res,
                   long res_stride, const void* weight, bool weight_f32,
                   float eps, void* h, void* y, int R, int K,
                   hipStream_t stream) {
  return by_type<false>(t, NormArgs{x, res, weight, h, y, nullptr, x_stride,
                                    res_stride, R, K, 0, eps, weight_f32},
                        stream);
}

hipError_t rmsnorm_mx(ActType t, const void* x, long x_stride, const void* res,
                      long res_stride, const void* weight, bool weight_f32,
                      float eps, void* h, unsigned char* q, unsigned char* sc,
                      int R, int K, hipStream_t stream) {
  return by_type<true>(t, NormArgs{x, res, weight, h, q, sc, x_stride,
                                   res_stride, R, K, 0, eps, weight_f32},
                       stream);
}

}  // namespace lpx
