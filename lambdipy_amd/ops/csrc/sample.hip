// One token for each row of logits: temperature, top-k, top-p, min-p and the
// draw, from a given uniform number.
//
//   w_i = exp((x_i - max x) / T), the row in the order (x falling, i rising);
//   kept is a prefix of that order: the shortest of the first k, of the
//   shortest one holding a share p of those k's weight, and of w_i >= min_p;
//   the token is the first whose running weight exceeds u times the kept.
//
// All three filters and the draw ask the same thing of the sorted row: where
// does a running count or a running weight pass a border. Nothing is sorted
// for that. Weights are 64-bit integers (w_i * 2^45, rounded), so that their
// sums do not depend on the order of adding: a border in a flat row of 10^5
// logits is decided by the 10th digit of a sum.
//
// 16-bit rows: one workgroup a row counts each of the 65536 values in LDS and
// looks the borders up among them; the exps are as many as the values that
// occur. 256 x 131072 bf16: 33 us, 32 where 9 of 10 are masked, 14 greedy; of
// the 26 in the kernel the LDS atomics of the counting take 11, reading the
// row a second time for the index 5, the sums and exps of its 72 groups of 64
// values 4 (with top-k fewer of them). 1 x 32000: 15 us, with top-k 14; 1 x
// 524288: 64 (115 as f32).
//
// f32 rows: a histogram of 256 bins, linear in x below the maximum, tells the
// bin that holds a border, and only that bin's members are looked at. An exp
// a logit in 64 bits, some 36 instructions, is what that takes; the instructions
// bound it. Short rows in one workgroup each; long ones as chunks (maxima,
// then histograms) and one workgroup a row for the borders: 24 x 50001 26 us,
// 256 x 131072 94 us, 99 from memory.

#include "lpx_common.h"
#include "kernels.h"

namespace lpx {

namespace {

typedef unsigned long long u64;

constexpr int BINS = 256;
constexpr int CHUNK_THREADS = 256;
constexpr int ROW_THREADS = 1024;
constexpr int LIST = 512;   // members of bins that a wave keeps in LDS
constexpr int FEW = 64;     // members that one wave ranks
// f32 rows up to here are one workgroup's, by measured time: one row of 16000
// takes 16 us so and 19 as chunks, of 32000 24 and 22; 256 rows of 32000 29
// and 40, of 64000 48 and 58.
constexpr int WHOLE = 24576, WHOLE_MANY = 65536, MANY = 96;

struct ChunkMax {
  float hi, lo;  // largest; smallest that is not -inf
  int at;        // lowest index of the largest
};

struct ChunkBins {
  u64 mass[BINS];
  unsigned count[BINS];
  u64 minp;  // mass of w >= min_p
};

struct RowScale {
  float hi;       // the row's largest logit
  float per_bin;  // bins per unit of x
  double hi64;    // a number over f32's where that is infinite
  double per_x;   // powers of two per unit of x
  double shift;
  int at;
  bool greedy, by_k, by_p;
};

struct SampleArgs {
  const void* logits;
  long stride;  // elements
  int rows, vocab, chunk, chunks, shift;
  SampleParam temperature, top_k, top_p, min_p, u;
  ChunkMax* maxima;  // [rows][chunks]
  ChunkBins* bins;   // [rows][chunks]
  RowScale* scales;  // [rows]
  bool binned;       // the last two are there
  int64_t* token;
};

__device__ __forceinline__ double param(const SampleParam& p, int row) {
  switch (p.kind) {
    case SampleParam::f32: return static_cast<const float*>(p.ptr)[row];
    case SampleParam::f64: return static_cast<const double*>(p.ptr)[row];
    case SampleParam::i32: return static_cast<const int*>(p.ptr)[row];
    case SampleParam::i64: return (double)static_cast<const int64_t*>(p.ptr)[row];
    default: return p.value;
  }
}

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float as_f32(__bf16 x) { return (float)x; }

// Bytes of a load. 16-bit rows come here seldom, and their kernel has no
// registers for more.
template <typename T>
constexpr int LOAD = sizeof(T) == 2 ? 4 : 16;

// f(index, logit) for every logit of [begin, end). A thread's indices rise.
// AHEAD: loads in flight a thread.
template <int THREADS, int AHEAD, typename T, typename F>
__device__ __forceinline__ void scan(const T* __restrict__ row, int begin,
                                     int end, F f) {
  constexpr int VEC = LOAD<T> / sizeof(T);
  typedef T V __attribute__((ext_vector_type(VEC)));
  const int tid = (int)threadIdx.x;
  const int off = (int)((uintptr_t)(row + begin) % LOAD<T> / sizeof(T));
  const int head = min(off ? VEC - off : 0, end - begin);
  if (tid < head) f(begin + tid, as_f32(row[begin + tid]));
  const int first = begin + head;
  const int vecs = (end - first) / VEC;
  const V* body = reinterpret_cast<const V*>(row + first);
  for (int i = tid; i < vecs; i += AHEAD * THREADS) {
    V v[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      if (i + a * THREADS < vecs) v[a] = body[i + a * THREADS];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a * THREADS >= vecs) break;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        f(first + (i + a * THREADS) * VEC + j, as_f32(v[a][j]));
    }
  }
  const int tail = first + vecs * VEC + tid;
  if (tail < end) f(tail, as_f32(row[tail]));
}

// Over the wave's lanes by DPP, not through LDS: what a lane takes from lanes
// below it (0 where there are none).
#define LPX_FROM(v, ctrl, rows) \
  (unsigned)__builtin_amdgcn_update_dpp(0, (int)(v), ctrl, rows, 0xf, false)
#define LPX_ROW_STEPS(STEP) /* row_shr 1, 2, 4, 8: within 16 lanes */ \
  STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf)
#define LPX_SIX_STEPS(STEP) /* and row_bcast 15 and 31 */ \
  LPX_ROW_STEPS(STEP) STEP(0x142, 0xa) STEP(0x143, 0xc)
#define LPX_ADD_64(ctrl, rows)                            \
  {                                                       \
    const unsigned lo = LPX_FROM((unsigned)v, ctrl, rows); \
    v += (u64)LPX_FROM(v >> 32, ctrl, rows) << 32 | lo;    \
  }
#define LPX_ADD_32(ctrl, rows) v += LPX_FROM(v, ctrl, rows);
#define LPX_MAX_32(ctrl, rows) v = max(v, LPX_FROM(v, ctrl, rows));

// Running sums, of 16 lanes and of all.
__device__ __forceinline__ unsigned row_run_up(unsigned v) {
  LPX_ROW_STEPS(LPX_ADD_32)
  return v;
}
__device__ __forceinline__ u64 wave_run_up(u64 v) {
  LPX_SIX_STEPS(LPX_ADD_64)
  return v;
}
__device__ __forceinline__ unsigned wave_run_up(unsigned v) {
  LPX_SIX_STEPS(LPX_ADD_32)
  return v;
}

// Bits of 16 lanes, to the last of them.
__device__ __forceinline__ unsigned row_or(unsigned v) {
#define LPX_OR_32(ctrl, rows) v |= LPX_FROM(v, ctrl, rows);
  LPX_ROW_STEPS(LPX_OR_32)
  return v;
}

// The largest, to every lane.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
  LPX_SIX_STEPS(LPX_MAX_32)
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// ---- a row's weights and bins --------------------------------------------

// A token can be drawn from this logit: it is not -inf and not NaN.
__device__ __forceinline__ bool real(float x) { return x > -__builtin_inff(); }

// The largest logit with its lowest index, and the smallest.
struct Extent {
  float hi = -__builtin_inff(), lo = __builtin_inff();
  int at = 0x7fffffff;
  __device__ __forceinline__ void join(float h, float l, int i) {
    if (h > hi || (h == hi && i < at)) {
      hi = h;
      at = i;
    }
    lo = fminf(lo, l);
  }
  __device__ __forceinline__ void join_wave() {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1)
      join(__shfl_xor(hi, m, 64), __shfl_xor(lo, m, 64), __shfl_xor(at, m, 64));
  }
};

constexpr double INFINITE = 1e300;

__device__ __forceinline__ RowScale row_scale(const SampleArgs& a, int row,
                                              Extent e) {
#pragma clang fp contract(off)
  RowScale r;
  r.hi = e.hi;
  r.hi64 = fmin((double)e.hi, INFINITE);
  r.at = e.hi > -__builtin_inff() ? e.at : -1;
  const double t = param(a.temperature, row);
  r.greedy = !(t > 0) || r.at < 0;
  r.by_k = param(a.top_k, row) >= 1;
  r.by_p = param(a.top_p, row) < 1;
  // 1 / (T ln 2); beside +inf a finite logit weighs nothing at any T
  r.per_x = e.hi == __builtin_inff() ? 1.0 : fmin(1.4426950408889634 / t, 1e300);
  r.shift = a.shift;
  // Below 32 T the weight rounds to nothing (e^-32 < 2^-46). A range that is
  // nothing or infinite is one bin.
  const double reach = fmin((double)e.hi - (double)e.lo, 32.0 * t);
  const double per = BINS / reach;
  r.per_bin = !(reach > 0) || e.hi == __builtin_inff() ? 0.f
              : per < 1e30                             ? (float)per
                                                       : 1e30f;
  return r;
}

// The row's extent from its chunks': every wave works it out for itself.
// `own`: the lane's, or the last.
__device__ __forceinline__ Extent row_extent(const SampleArgs& a, int row,
                                             ChunkMax own) {
  const ChunkMax* c = a.maxima + (long)row * a.chunks;
  Extent e;
  e.join(own.hi, own.lo, own.at);
  for (int i = 64 + ((int)threadIdx.x & 63); i < a.chunks; i += 64)
    e.join(c[i].hi, c[i].lo, c[i].at);
  e.join_wave();
  return e;
}

__device__ __forceinline__ int bin_of(const RowScale& r, float x) {
#pragma clang fp contract(off)
  // falls as x rises; 0 * inf ends in the last bin
  return (int)fminf((r.hi - x) * r.per_bin, (float)(BINS - 1));
}

// a * b + c in one instruction. (From the builtin the compiler makes the
// two-address form and a move for every constant.)
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
  return d;
}

// 2^shift * exp((x - hi) / T), rounded; 0 of -inf and NaN. The same bits
// wherever it is inlined: nothing here is contracted in one place and not in
// another.
__device__ __forceinline__ u64 weight(const RowScale& r, float x) {
#pragma clang fp contract(off)
  // NaN becomes -inf here: left to the arithmetic it is +inf, as fmin takes
  // the number of the two
  const double d = fmin((double)(real(x) ? x : -__builtin_inff()), INFINITE) - r.hi64;
  // 2^-2 and less rounds to nothing; so does -inf at an infinite T, where the
  // product is NaN
  const double y = fmax(__builtin_fma(d, r.per_x, r.shift), -2.0);
  const double n = __builtin_rint(y), f = y - n;
  // (2^f - 1) / f on [-1/2, 1/2], the polynomial of degree 8 through nine
  // Chebyshev nodes: 2^f is off by 2^-44.6 of itself at most
  double p = 1.0203121156603192e-07;
  p = fma_const(f, p, 1.325522487537687e-06);
  p = fma_const(p, f, 1.5252686845879443e-05);
  p = fma_const(p, f, 0.0001540345585246757);
  p = fma_const(p, f, 0.001333355817904356);
  p = fma_const(p, f, 0.009618129159402543);
  p = fma_const(p, f, 0.055504108664760424);
  p = fma_const(p, f, 0.2402265069581299);
  p = fma_const(p, f, 0.6931471805599453);
  p = fma_const(p, f, 1.0);
  // 2^52 more leaves the rounded integer in the low bits
  const double w = __builtin_amdgcn_ldexp(p, (int)n) + 0x1p52;
  return (u64)__builtin_bit_cast(long long, w) & 0xfffffffffffffull;
}

// The least weight that min-p keeps.
__device__ __forceinline__ u64 least_weight(const SampleArgs& a, int row,
                                            const RowScale& r) {
  const double p = fmax(0.0, fmin(param(a.min_p, row), 2.0));
  return (u64)ceil(p * (double)(1ll << (int)r.shift));
}

// What a running mass has to reach to hold a share of another; what it has to
// reach to exceed u times that.
__device__ __forceinline__ u64 share_of(double part, u64 of) {
  const double s = ceil(part * (double)of);
  return s >= (double)of ? of : s > 1 ? (u64)s : (u64)1;
}

__device__ __forceinline__ u64 draw_border(double u, u64 of) {
  const double s = floor(u * (double)of);
  return s >= (double)of ? max(of, (u64)1) : s > 0 ? (u64)s + 1 : (u64)1;
}

// ---- 1: maxima ------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(CHUNK_THREADS) void chunk_max_kernel(SampleArgs a) {
  const int row = (int)blockIdx.x / a.chunks;
  const int begin = (int)blockIdx.x % a.chunks * a.chunk;
  const int end = min(begin + a.chunk, a.vocab);
  Extent e;
  scan<CHUNK_THREADS, 2>(static_cast<const T*>(a.logits) + row * a.stride, begin,
                         end, [&](int i, float x) {
                           e.join(x, real(x) ? x : e.lo, i);
                         });
  e.join_wave();
  __shared__ ChunkMax part[CHUNK_THREADS / 64];
  if ((threadIdx.x & 63) == 0)
    part[threadIdx.x >> 6] = ChunkMax{e.hi, e.lo, e.at};
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < CHUNK_THREADS / 64; ++i)
    e.join(part[i].hi, part[i].lo, part[i].at);
  a.maxima[blockIdx.x] = ChunkMax{e.hi, e.lo, e.at};
}

// ---- 2: histograms --------------------------------------------------------

// Adds [begin, end) of a row to bins in LDS: the logits that have a weight.
// (The others follow them all, and cutting among those changes nothing. Where
// a mask is the type's lowest value they are most of a row, in one bin.)
// Counts are only asked for where the row is cut by top-k or top-p.
template <int THREADS, typename T, typename B>
__device__ __forceinline__ void add_bins(B& b, const RowScale& r, u64 least,
                                         const T* row, int begin, int end) {
  const bool counted = r.by_k || r.by_p;
  u64 minp = 0;
  scan<THREADS, 2>(row, begin, end, [&](int, float x) {
    const int bin = bin_of(r, x);
    const u64 w = weight(r, x);
    if (w) {
      if (counted) atomicAdd(&b.count[bin], 1u);
      atomicAdd(&b.mass[bin], w);
    }
    minp += w >= least ? w : 0;
  });
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) minp += __shfl_xor(minp, m, 64);
  if ((threadIdx.x & 63) == 0) atomicAdd(&b.minp, minp);
}

template <typename T>
__global__ __launch_bounds__(CHUNK_THREADS) void chunk_bins_kernel(SampleArgs a) {
  const int row = (int)blockIdx.x / a.chunks;
  const int begin = (int)blockIdx.x % a.chunks * a.chunk;
  const int end = min(begin + a.chunk, a.vocab);
  const ChunkMax* maxima = a.maxima + (long)row * a.chunks;
  const ChunkMax own = maxima[min((int)threadIdx.x & 63, a.chunks - 1)];
  const RowScale r = row_scale(a, row, row_extent(a, row, own));
  if (begin == 0 && threadIdx.x == 0) a.scales[row] = r;
  if (r.greedy) return;
  __shared__ ChunkBins b;
  b.mass[threadIdx.x] = 0;
  b.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) b.minp = 0;
  __syncthreads();
  add_bins<CHUNK_THREADS>(b, r, least_weight(a, row, r),
                          static_cast<const T*>(a.logits) + row * a.stride, begin, end);
  __syncthreads();
  ChunkBins& out = a.bins[blockIdx.x];
  out.mass[threadIdx.x] = b.mass[threadIdx.x];
  out.count[threadIdx.x] = b.count[threadIdx.x];
  if (threadIdx.x == 0) out.minp = b.minp;
}

// ---- 3: borders -----------------------------------------------------------

// Sorts ascending as (x falling, index rising); no two are equal.
__device__ __forceinline__ u64 order_of(float x, int i) {
  const unsigned b = __float_as_uint(x + 0.f);  // -0 is 0
  const unsigned up = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((u64)~up << 32) | (unsigned)i;
}

__device__ __forceinline__ float logit_of(u64 o) {
  const unsigned up = ~(unsigned)(o >> 32);
  return __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
}

// The lowest logit in bin `bin` or above, which is where the bin begins. The
// wave looks at 64 of f32's values at a time, in the order of their bits.
__device__ __forceinline__ float bin_begin(const RowScale& r, int bin) {
  const auto up = [](float x) { return ~(unsigned)(order_of(x, 0) >> 32); };
  const unsigned most = up(r.hi), least = up(-3.402823466e38f);
  unsigned at = 0;
#pragma unroll 1
  for (int shift = 26; shift >= -4; shift -= 6) {
    const int s = max(shift, 0);
    const unsigned lane = threadIdx.x & 63;
    const unsigned last = at + (lane << s) + ((1u << s) - 1);
    const bool over = last < at;  // past the highest bits
    const unsigned key = over ? most : max(min(last, most), least);
    const u64 in = __ballot(bin_of(r, logit_of((u64)~key << 32)) <= bin);
    at += (unsigned)__builtin_ctzll(in) << s;
  }
  return logit_of((u64)~max(min(at, most), least) << 32);
}

struct Member {
  u64 order, weight;
};

struct RowShared {
  ChunkBins row, sub;  // running sums, bin by bin
  u64 list[ROW_THREADS / 64][LIST];
  int listed[ROW_THREADS / 64];
  Member few[FEW];
  ChunkMax extent[ROW_THREADS / 64];
  u64 wave_mass[BINS / 64];
  unsigned wave_count[BINS / 64];
  u64 lo, hi;
  int bin, found;
  u64 mass;  // a border's answer
  int at;
};

__device__ __forceinline__ void clear(ChunkBins& b) {
  if (threadIdx.x < BINS) {
    b.mass[threadIdx.x] = 0;
    b.count[threadIdx.x] = 0;
  }
  if (threadIdx.x == 0) b.minp = 0;
}

// Counts and masses of bins -> running sums.
__device__ __forceinline__ void run_up(ChunkBins& b, RowShared& sh) {
  const int t = (int)threadIdx.x, lane = t & 63;
  u64 m = 0;
  unsigned c = 0;
  if (t < BINS) {
    m = wave_run_up(b.mass[t]);
    c = wave_run_up(b.count[t]);
    if (lane == 63) {
      sh.wave_mass[t >> 6] = m;
      sh.wave_count[t >> 6] = c;
    }
  }
  __syncthreads();
  if (t < BINS) {
    for (int w = 0; w < (t >> 6); ++w) {
      m += sh.wave_mass[w];
      c += sh.wave_count[w];
    }
    b.mass[t] = m;
    b.count[t] = c;
  }
  if (t == 0) sh.bin = BINS - 1;
  __syncthreads();
}

// The first bin whose running sum reaches `border`, which some bin's does.
// (One thread at most writes sh.bin; it holds some bin from run_up on.)
__device__ __forceinline__ int bin_at(const ChunkBins& b, bool by_count,
                                      u64 border, RowShared& sh) {
  const int t = (int)threadIdx.x;
  if (t < BINS) {
    const u64 now = by_count ? b.count[t] : b.mass[t];
    const u64 before = t == 0 ? 0 : by_count ? b.count[t - 1] : b.mass[t - 1];
    if (now >= border && before < border) sh.bin = t;
  }
  __syncthreads();
  const int bin = sh.bin;
  __syncthreads();
  return bin;
}

template <typename T>
struct RowPick {
  const SampleArgs& a;
  const T* row;
  const RowScale r;
  RowShared& sh;
  int first = 0, last = -1;  // the bins whose members are in the lists
  unsigned found = 0;        // and how many they are

  __device__ __forceinline__ bool listed(int bin) const {
    return first <= bin && bin <= last;
  }

  // f(order, logit) of the members of `bin` between lo and hi
  template <typename F>
  __device__ __forceinline__ void members(int bin, u64 lo, u64 hi, F f) {
    if (listed(bin)) {
      const int wave = (int)threadIdx.x >> 6, n = sh.listed[wave];
      for (int i = (int)threadIdx.x & 63; i < n; i += 64) {
        const u64 o = sh.list[wave][i];
        const float x = logit_of(o);
        if (bin_of(r, x) == bin && lo <= o && o <= hi) f(o, x);
      }
    } else {
      scan<ROW_THREADS, 1>(row, 0, a.vocab, [&](int i, float x) {
        if (bin_of(r, x) != bin || !real(x)) return;
        const u64 o = order_of(x, i);
        if (lo <= o && o <= hi) f(o, x);
      });
    }
  }

  // Lists the members of bins [from, to], unless a wave's are too many.
  __device__ __forceinline__ void collect(int from, int to) {
    constexpr int VEC = LOAD<T> / sizeof(T), AHEAD = 4;
    typedef T V __attribute__((ext_vector_type(VEC)));
    // the bins as an interval, so that a logit takes two comparisons
    const float low = bin_begin(r, to);
    const float high = bin_of(r, r.hi) < from
                           ? logit_of(order_of(bin_begin(r, from - 1), 0) + (1ull << 32))
                           : __builtin_inff();  // the next lower logit
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // Each wave has a list of its own and knows its length: no atomic, whose
    // answer would have to be waited for. First of indices: a lane has a bit
    // for each of its logits.
    int have = 0;
    u64* list = sh.list[wave];
    auto in = [&](float x) { return __builtin_amdgcn_fmed3f(x, low, high) == x; };
    auto add = [&](unsigned bits, auto index) {
      const unsigned n = (unsigned)__popc(bits), up = wave_run_up(n);
      for (unsigned at = have + up - n; bits; bits &= bits - 1, ++at)
        if (at < LIST) list[at] = (unsigned)index(__builtin_ctz(bits));
      have += __builtin_amdgcn_readlane((int)up, 63);
    };
    const int off = (int)((uintptr_t)row % LOAD<T> / sizeof(T));
    const int head = min(off ? VEC - off : 0, a.vocab);
    const int vecs = (a.vocab - head) / VEC;
    const V* body = reinterpret_cast<const V*>(row + head);
    if (wave == 0) {
      const int tail = head + vecs * VEC + lane;
      const unsigned first = lane < head && in(as_f32(row[lane]));
      const unsigned last = tail < a.vocab && in(as_f32(row[tail]));
      add(first | last << 1, [&](int bit) { return bit ? tail : lane; });
    }
    for (int v0 = wave * 64; v0 < vecs; v0 += AHEAD * ROW_THREADS) {
      V v[AHEAD];
#pragma unroll
      for (int l = 0; l < AHEAD; ++l)
        v[l] = body[min(v0 + l * ROW_THREADS + lane, vecs - 1)];
      unsigned bits = 0;
#pragma unroll
      for (int l = 0; l < AHEAD; ++l)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          bits |= (unsigned)in(as_f32(v[l][j])) << (l * VEC + j);
      // those behind the row's end
      const int left = vecs - v0 - lane;
      if (left <= (AHEAD - 1) * ROW_THREADS) {
        const int whole = left <= 0 ? 0 : (left + ROW_THREADS - 1) / ROW_THREADS;
        bits &= (1u << (whole * VEC)) - 1;
      }
      if (__ballot(bits != 0))
        add(bits, [&](int bit) {
          return head + (v0 + bit / VEC * ROW_THREADS + lane) * VEC + bit % VEC;
        });
    }
    // then of places in the order
    for (int i = lane; i < min(have, LIST); i += 64) {
      const int at = (int)list[i];
      list[i] = order_of(as_f32(row[at]), at);
    }
    if (lane == 0) sh.listed[wave] = have;
    __syncthreads();
    unsigned all = 0;
    bool fits = true;
    for (int w = 0; w < ROW_THREADS / 64; ++w) {
      const int n = sh.listed[w];
      all += n;
      fits &= n <= LIST;
    }
    first = from;
    last = fits ? to : from - 1;
    found = all;
  }

  // The member of the row at which the running count (mass) reaches `border`:
  // its index to sh.at, the running mass with it to sh.mass. `more`: borders
  // further up will be asked for, so that all from the top is listed if it
  // fits.
  __device__ __forceinline__ void resolve(bool by_count, u64 border, bool more) {
    const int bin = bin_at(sh.row, by_count, border, sh);
    // what stands before [lo, hi], and how many members that has at most
    unsigned base = bin ? sh.row.count[bin - 1] : 0;
    u64 mass = bin ? sh.row.mass[bin - 1] : 0;
    for (int from = more && sh.row.count[bin] <= LIST * 8 ? 0 : bin; !listed(bin);) {
      collect(from, bin);
      if (from == bin) break;
      from = bin;  // that alone, if all does not fit
      __syncthreads();
    }
    // (bins are counted where more than one is listed)
    unsigned n = first == bin && (last == bin || !listed(bin)) ? found
                                                               : sh.row.count[bin] - base;
    u64 lo = 0, hi = ~0ull;
    while (n > FEW) {
      // 256 sub-bins between the first and the last member; the two differ,
      // so that n falls with every turn
      if (threadIdx.x == 0) {
        sh.lo = ~0ull;
        sh.hi = 0;
      }
      clear(sh.sub);
      __syncthreads();
      u64 tlo = ~0ull, thi = 0;
      members(bin, lo, hi, [&](u64 o, float) {
        tlo = min(tlo, o);
        thi = max(thi, o);
      });
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) {
        tlo = min(tlo, (u64)__shfl_xor(tlo, m, 64));
        thi = max(thi, (u64)__shfl_xor(thi, m, 64));
      }
      if ((threadIdx.x & 63) == 0 && tlo <= thi) {
        atomicMin(&sh.lo, tlo);
        atomicMax(&sh.hi, thi);
      }
      __syncthreads();
      lo = sh.lo;
      hi = sh.hi;
      const int drop = max(0, 64 - __clzll((long long)(hi - lo)) - 8);
      members(bin, lo, hi, [&](u64 o, float x) {
        const int s = (int)((o - lo) >> drop);
        const u64 w = weight(r, x);
        if (!w) return;
        atomicAdd(&sh.sub.count[s], 1u);
        atomicAdd(&sh.sub.mass[s], w);
      });
      __syncthreads();
      run_up(sh.sub, sh);
      const int s = bin_at(sh.sub, by_count, border - (by_count ? base : mass), sh);
      const unsigned before = s ? sh.sub.count[s - 1] : 0;
      n = sh.sub.count[s] - before;
      base += before;
      mass += s ? sh.sub.mass[s - 1] : 0;
      lo += (u64)s << drop;
      hi = lo + min(hi - lo, (1ull << drop) - 1);
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      sh.found = 0;
      sh.at = r.at;
      sh.mass = mass;
    }
    __syncthreads();
    members(bin, lo, hi, [&](u64 o, float x) {
      const u64 w = weight(r, x);
      if (!w) return;
      const int i = atomicAdd(&sh.found, 1);
      if (i < FEW) sh.few[i] = Member{o, w};
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      // each lane adds up what is before its member
      const unsigned found = min(sh.found, FEW);
      const bool mine = threadIdx.x < found;
      const Member own = sh.few[mine ? threadIdx.x : 0];
      unsigned before = 0;
      u64 run = 0;
      for (unsigned j = 0; j < found; ++j) {
        const Member other = sh.few[j];
        const bool less = other.order < own.order;
        before += less;
        run += less ? other.weight : 0;
      }
      const u64 was = by_count ? base + before : mass + run;
      const u64 now = was + (by_count ? 1 : own.weight);
      if (mine && now >= border && was < border) {
        sh.mass = mass + run + own.weight;
        sh.at = (int)(unsigned)own.order;
      }
    }
    __syncthreads();
  }
};

// The borders of a row whose running sums are in sh.row.
template <typename T>
__device__ __forceinline__ int pick_token(const SampleArgs& a, int row,
                                          const RowScale& r, RowShared& sh) {
  const u64 total = sh.row.mass[BINS - 1];
  const unsigned all = sh.row.count[BINS - 1];
  RowPick<T> pick{a, static_cast<const T*>(a.logits) + row * a.stride, r, sh};

  u64 kept = total;
  const double k = param(a.top_k, row);
#pragma unroll 1  // one copy of the code for the three borders
  for (int cut = 0; cut < 3; ++cut) {
    u64 border;
    if (cut == 0) {
      if (!(r.by_k && k < (double)all)) continue;
      border = (u64)k;
    } else if (cut == 1) {
      if (!r.by_p) continue;
      border = share_of(param(a.top_p, row), kept);
    } else {
      border = draw_border(param(a.u, row), min(kept, sh.row.minp));
    }
    pick.resolve(cut == 0, border, cut < 2);
    kept = sh.mass;
  }
  return sh.at;
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void row_pick_kernel(SampleArgs a) {
  __shared__ RowShared sh;
  const int row = (int)blockIdx.x, t = (int)threadIdx.x;
  if (!a.binned) {  // greedy, as the host knows
    const ChunkMax* maxima = a.maxima + (long)row * a.chunks;
    const Extent e = row_extent(a, row, maxima[min(t & 63, a.chunks - 1)]);
    if (t == 0) a.token[row] = row_scale(a, row, e).at;
    return;
  }
  const RowScale r = a.scales[row];
  // thread t sums bin t % BINS over a quarter of the chunks
  const ChunkBins* c = a.bins + (long)row * a.chunks;
  const int bin = t % BINS;
  u64 m = 0, minp = 0;
  unsigned n = 0;
  for (int i0 = t / BINS; i0 < a.chunks; i0 += 4 * (ROW_THREADS / BINS)) {
    u64 mass[4], least[4];
    unsigned count[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // all on their way at once
      const ChunkBins& b = c[min(i0 + j * (ROW_THREADS / BINS), a.chunks - 1)];
      mass[j] = b.mass[bin];
      count[j] = b.count[bin];
      least[j] = b.minp;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j * (ROW_THREADS / BINS) >= a.chunks) break;
      m += mass[j];
      n += count[j];
      minp += least[j];
    }
  }
  clear(sh.row);
  if (r.greedy) {
    if (t == 0) a.token[row] = r.at;
    return;
  }
  __syncthreads();
  atomicAdd(&sh.row.mass[bin], m);
  atomicAdd(&sh.row.count[bin], n);
  if (bin == 0) atomicAdd(&sh.row.minp, minp);
  __syncthreads();
  run_up(sh.row, sh);
  const int token = pick_token<T>(a, row, r, sh);
  if (t == 0) a.token[row] = token;
}

// All of a row in one workgroup.
template <typename T>
__device__ __forceinline__ void whole_row(const SampleArgs& a, int row, RowShared& sh) {
  const int t = (int)threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  Extent e;
  scan<ROW_THREADS, 4>(x, 0, a.vocab, [&](int i, float v) {
    e.join(v, real(v) ? v : e.lo, i);
  });
  e.join_wave();
  if ((t & 63) == 0) sh.extent[t >> 6] = ChunkMax{e.hi, e.lo, e.at};
  clear(sh.row);
  __syncthreads();
  {
    const ChunkMax c = sh.extent[t & (ROW_THREADS / 64 - 1)];
    e.join(c.hi, c.lo, c.at);
    e.join_wave();
  }
  const RowScale r = row_scale(a, row, e);
  if (r.greedy) {
    if (t == 0) a.token[row] = r.at;
    return;
  }
  add_bins<ROW_THREADS>(sh.row, r, least_weight(a, row, r), x, 0, a.vocab);
  __syncthreads();
  run_up(sh.row, sh);
  const int token = pick_token<T>(a, row, r, sh);
  if (t == 0) a.token[row] = token;
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void row_whole_kernel(SampleArgs a) {
  __shared__ RowShared sh;
  whole_row<T>(a, (int)blockIdx.x, sh);
}

// ---- 16-bit rows ----------------------------------------------------------
// There are 65536 logits of 16 bits, so a row is the count of each: one LDS
// atomic a logit, and an exp for each of the few thousand values that occur.
// The borders are then looked up among the values, and where equal logits
// stand on one, the row is read once more for the index of the one meant.
//
// A value's place is its rank from the top: positive ones 0x7fff - bits,
// negative ones their bits. Ranks below that of +inf are NaN, those from
// that of -inf on are -inf and NaN.

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int GROUPS = 1024;  // of 64 neighbouring ranks
constexpr unsigned MANY_COPIES = 64;  // of a value; fewer are listed
static_assert(SAMPLE_MOST_16 == GROUPS * 512, "a row's counts of 512 logits");

template <typename T> struct Ranks;
template <> struct Ranks<__bf16> {
  static constexpr unsigned INF = 0x7fff - 0x7f80, NONE = 0xff80;
  static __device__ __forceinline__ float value(unsigned bits) {
    return __uint_as_float(bits << 16);
  }
};
template <> struct Ranks<_Float16> {
  static constexpr unsigned INF = 0x7fff - 0x7c00, NONE = 0xfc00;
  static __device__ __forceinline__ float value(unsigned bits) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
  }
};

// Bits to rank and back; two values at once.
__device__ __forceinline__ unsigned ranks_of(unsigned two) {
  const unsigned positive = ~two & 0x80008000u;
  return two ^ (positive - (positive >> 15));
}

struct TableShared {
  // Rank r's count is in half r >> 15 of word r & 0x7fff. A count of 65536
  // and more runs over; the counts' sum then falls short of the row's length.
  // A lowest value that is often there, a mask's say, has a count of its own.
  unsigned count[32768];
  unsigned last, lowest;   // that value's rank (0: none) and count
  u64 mass[GROUPS];        // of 64 ranks; running sums later
  unsigned members[GROUPS];  // counted for top-k; later for 512 logits each
  u64 wave_mass[ROW_THREADS / 64];
  unsigned wave_members[ROW_THREADS / 64];
  unsigned first;          // the highest logit's rank
  unsigned logits;
  u64 minp;
  int group;
  unsigned rank, copy;     // a border's answer: its value, which of equal ones
  unsigned listed, list[MANY_COPIES];  // those
  int lowest_at;           // greedy: the token
  unsigned groups;         // that hold something
  unsigned short group_list[GROUPS];
  u64 kept;                // and the running mass with it
  int token;
};

template <typename T>
__device__ __forceinline__ float logit_at(unsigned rank) {
  return Ranks<T>::value((rank >> 15 ? rank : 0x7fffu - rank) & 0xffffu);
}

__device__ __forceinline__ unsigned count_at(const TableShared& sh, unsigned rank) {
  if (rank == sh.last) return sh.lowest;
  return (sh.count[rank & 0x7fff] >> (rank >> 15 ? 16 : 0)) & 0xffffu;
}

// The value at which the running count (mass) reaches `border`, which of its
// copies does, and the running mass with that.
template <typename T>
__device__ __forceinline__ void find_border(TableShared& sh, const RowScale& r,
                                            bool by_count, u64 border) {
  const int t = (int)threadIdx.x;
  {
    const u64 now = by_count ? sh.members[t] : sh.mass[t];
    const u64 before = t == 0 ? 0 : by_count ? sh.members[t - 1] : sh.mass[t - 1];
    if (now >= border && before < border) sh.group = t;
  }
  __syncthreads();
  if (t < 64) {
    const int group = sh.group;
    const unsigned rank = (unsigned)group * 64 + t;
    const bool some = rank >= Ranks<T>::INF && rank < Ranks<T>::NONE;
    const u64 n = some ? count_at(sh, rank) : 0;
    const u64 w = n ? weight(r, logit_at<T>(rank)) : 0;
    // before this value
    const u64 mass = (group ? sh.mass[group - 1] : 0) + wave_run_up(n * w) - n * w;
    const u64 members =
        by_count ? (group ? sh.members[group - 1] : 0) + wave_run_up((unsigned)n) - n : 0;
    const u64 was = by_count ? members : mass, each = by_count ? 1 : w;
    if (was < border && was + n * each >= border) {
      // how many copies reach it: border - was of `each`, rounded up
      u64 need = border - was;
      if (!by_count) {
        // an estimate (at most 2^19 copies), put right
        u64 q = (u64)((float)need * __builtin_amdgcn_rcpf((float)w));
        while (q * w < need) ++q;
        while (q > 1 && (q - 1) * w >= need) --q;
        need = q;
      }
      sh.rank = rank;
      sh.copy = (unsigned)need - 1;
      sh.kept = mass + need * w;
    }
  }
  __syncthreads();
}

// Running sums over the workgroup's threads.
template <typename N>
__device__ __forceinline__ N block_run_up(N v, N* waves) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  v = wave_run_up(v);
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  const N up = wave_run_up(lane < ROW_THREADS / 64 ? waves[lane] : (N)0);
  const N before = __shfl(up, max(wave - 1, 0), 64);
  return wave ? v + before : v;
}

// The logits of one value among a row's words.
struct Wanted {
  unsigned both, keep;
  __device__ __forceinline__ explicit Wanted(unsigned rank) {
    const unsigned bits = rank >> 15 ? rank : 0x7fffu - rank;
    both = bits << 16 | bits;
    keep = bits ? 0xffffffffu : 0x7fff7fffu;  // -0 is 0
  }
  // 0 for a logit that is it
  __device__ __forceinline__ u16x2 differ(int two) const {
    return __builtin_bit_cast(u16x2, ((unsigned)two & keep) ^ both);
  }
  __device__ __forceinline__ bool among(i32x4 v) const {
    const u16x2 d = __builtin_elementwise_min(
        __builtin_elementwise_min(differ(v[0]), differ(v[1])),
        __builtin_elementwise_min(differ(v[2]), differ(v[3])));
    return !d[0] || !d[1];
  }
  __device__ __forceinline__ unsigned copies(i32x4 v) const {
    u16x2 d = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      d += __builtin_elementwise_min(differ(v[j]), u16x2{1, 1});
    return 8u - d[0] - d[1];
  }
};

// The index of copy number `copy` of a value: the copies in every 512 logits
// are counted, and those that hold the one meant looked at again.
__device__ __forceinline__ int index_of(TableShared& sh, const unsigned short* row,
                                        int n, unsigned rank, unsigned copy) {
  const int t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  constexpr int WAVES = ROW_THREADS / 64;
  const Wanted wanted(rank);
  auto load = [&](int at) {
    i32x4 v;
    if (at + 8 <= n) {
      __builtin_memcpy(&v, row + at, 16);
    } else {  // what is not there is not it
      unsigned short w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        w[j] = at + j < n ? row[at + j] : (unsigned short)(wanted.both ^ 0x4000u);
      __builtin_memcpy(&v, w, 16);
    }
    return v;
  };
  sh.members[t] = 0;
  __syncthreads();
  const int blocks = (n + 511) / 512;  // GROUPS at most
  for (int b = wave; b < blocks; b += 4 * WAVES) {
    i32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (b + j * WAVES < blocks) v[j] = load((b + j * WAVES) * 512 + lane * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (b + j * WAVES >= blocks) break;
      const unsigned have = wanted.copies(v[j]);
      if (__ballot(have != 0)) {
        const unsigned all = wave_run_up(have);
        if (lane == 63) sh.members[b + j * WAVES] = all;
      }
    }
  }
  __syncthreads();
  const unsigned here = sh.members[t];
  const unsigned through = block_run_up(here, sh.wave_members);
  if (through - here <= copy && copy < through) {
    sh.group = t;
    sh.copy = copy - (through - here);
  }
  __syncthreads();
  if (wave == 0) {
    const int at = sh.group * 512 + lane * 8;
    const i32x4 v = load(at);
    const unsigned have = wanted.copies(v), up = wave_run_up(have);
    unsigned left = sh.copy - (up - have);
    if (up - have <= sh.copy && sh.copy < up) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u16x2 d = wanted.differ(v[j / 2]);
        if (!d[j % 2] && left-- == 0) sh.token = at + j;
      }
    }
  }
  __syncthreads();
  return sh.token;
}

template <typename T>
__global__ __launch_bounds__(ROW_THREADS) void row_table_kernel(SampleArgs a) {
  __shared__ union Shared {
    TableShared table;
    RowShared row;
    __device__ Shared() {}
  } shared;
  TableShared& sh = shared.table;
  const int row = (int)blockIdx.x, t = (int)threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const unsigned short* x = static_cast<const unsigned short*>(a.logits) + row * a.stride;
  const bool greedy = !(param(a.temperature, row) > 0);

  // The row: 16-B vectors, STEP at a time, and the elements at its ends, one
  // for each of 16 threads. The first loads go out before all else, and the
  // last ones' registers are kept for the search for the index.
  constexpr int AHEAD = 4, STEP = AHEAD * ROW_THREADS;
  const int vocab = a.vocab;
  const int off = (int)(((uintptr_t)x & 15) / 2);
  const int head = min(off ? 8 - off : 0, vocab);
  const int vecs = (vocab - head) / 8;
  const i32x4* body = reinterpret_cast<const i32x4*>(x + head);
  auto load = [&](i32x4* to, int first) {
#pragma unroll
    for (int l = 0; l < AHEAD; ++l)
      if (first + l * ROW_THREADS < vecs)
        to[l] = body[min(first + l * ROW_THREADS + lane, vecs - 1)];
  };
  int v0 = wave * 64;
  i32x4 v[AHEAD];
  load(v, v0);
  int edge = vocab;
  if (t < 16) edge = t < 8 ? (t < head ? t : vocab) : head + vecs * 8 + t - 8;
  const unsigned edge_bits = edge < vocab ? x[edge] : 0u;

  {
    const i32x4 zero = {0, 0, 0, 0};
    i32x4* words = reinterpret_cast<i32x4*>(sh.count);
    if (!greedy)
      for (int i = t; i < 8192; i += ROW_THREADS) words[i] = zero;
    sh.mass[t] = 0;
    sh.members[t] = 0;
    if (t == 0) {
      sh.first = 0xffffu;
      sh.last = 0;
      sh.lowest = 0;
      sh.logits = 0;
      sh.minp = 0;
      sh.group = 0;
      sh.rank = 0;
      sh.copy = 0;
      sh.kept = 0;
      sh.token = -1;
      sh.listed = 0;
      sh.groups = 0;
      sh.lowest_at = 0x7fffffff;
    }
  }
  __syncthreads();

  // Counts, and the highest: of ranks from +inf's on, of which NaN's are not.
  u16x2 lows = {0xffff, 0xffff};
  auto highest = [&](unsigned two) {
    const u16x2 above = __builtin_bit_cast(u16x2, two) -
                        u16x2{(unsigned short)Ranks<T>::INF, (unsigned short)Ranks<T>::INF};
    lows = __builtin_elementwise_min(lows, above);
  };
  auto add = [&](unsigned rank, unsigned n) {
    atomicAdd(&sh.count[rank & 0x7fff], n << (rank >> 15 << 4));
  };
  // Atomics on one word wait for each other: a masked row of 32000 took 37 us
  // by them. So where the lowest of the 2048 logits that a wave holds is in
  // many of its lanes, they count it in a register.
  unsigned last = 0, lowest = 0;
  constexpr int MANY_LANES = 8;
  if (!greedy && edge < vocab) add(ranks_of(edge_bits) & 0xffffu, 1u);
  unsigned best = 0xffffu;  // greedy: the lane's highest, and where it came first
  int best_at = 0;
  while (v0 < vecs) {
    const bool more = v0 + STEP < vecs;
    i32x4 next[AHEAD];
    if (more) load(next, v0 + STEP);
    u16x2 most = {0, 0};
#pragma unroll
    for (int l = 0; l < AHEAD; ++l) {
      if (v0 + l * ROW_THREADS >= vecs) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned two = ranks_of((unsigned)v[l][j]);
        highest(two);
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, two));
      }
    }
    if (greedy) {
      const unsigned now = min(lows[0], lows[1]);
      if (now < best) {
        best = now;
        best_at = v0;
      }
    } else {
      const unsigned own = min(max((unsigned)most[0], (unsigned)most[1]), Ranks<T>::NONE);
      const unsigned far = wave_max(own);
      const bool often = far >= last && __popcll(__ballot(own == far)) >= MANY_LANES;
      if (often && far > last) {
        if (lowest) add(last, lowest);
        last = far;
        lowest = 0;
      }
#pragma unroll
      for (int l = 0; l < AHEAD; ++l) {
        const int at = v0 + l * ROW_THREADS;
        if (at >= vecs) break;
        if (at + lane >= vecs) continue;
        if (often) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const unsigned rank = ranks_of((unsigned)v[l][j / 2]) >> (j % 2 * 16) & 0xffffu;
            if (rank == last)
              ++lowest;
            else
              add(rank, 1u);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            add(ranks_of((unsigned)v[l][j / 2]) >> (j % 2 * 16) & 0xffffu, 1u);
        }
      }
    }
    if (!more) break;
#pragma unroll
    for (int l = 0; l < AHEAD; ++l) v[l] = next[l];
    v0 += STEP;
  }
  if (edge < vocab) highest(ranks_of(edge_bits * 0x10001u));
  const unsigned low = 0xffffu - wave_max(0xffffu - min(lows[0], lows[1]));
  if (lane == 0) {
    atomicMin(&sh.first, low);
    atomicMax(&sh.last, last);
  }
  __syncthreads();
  unsigned first = sh.first + Ranks<T>::INF;
  if (first >= Ranks<T>::NONE) {  // nothing over -inf
    if (t == 0) a.token[row] = -1;
    return;
  }
  if (first == 0x8000u) first = 0x7fffu;
  if (greedy) {
    int token;
    if (first == 0x7fffu) {  // +0 and -0 are one
      token = index_of(sh, x, vocab, first, 0);
    } else {
      const Wanted wanted(first);
      int at = vocab;
      if (edge < vocab && !wanted.differ((int)edge_bits)[0]) at = edge;
      if (best == first - Ranks<T>::INF) {
        load(v, best_at);
#pragma unroll
        for (int l = AHEAD - 1; l >= 0; --l) {
          const int i = best_at + l * ROW_THREADS + lane;
          if (i >= vecs || !wanted.among(v[l])) continue;
#pragma unroll
          for (int j = 7; j >= 0; --j)
            if (!wanted.differ(v[l][j / 2])[j % 2]) at = min(at, head + i * 8 + j);
        }
      }
      if (at < vocab) atomicMin(&sh.lowest_at, at);
      __syncthreads();
      token = sh.lowest_at;
    }
    if (t == 0) a.token[row] = token;
    return;
  }
  {
    const unsigned n = wave_run_up(lowest);
    if (lane == 63 && n) {
      if (last == sh.last)
        atomicAdd(&sh.lowest, n);
      else
        add(last, n);
    }
  }
  __syncthreads();
  if (t == 0) {
    // -0 is 0
    const unsigned plus = sh.count[0x7fff] & 0xffffu, minus = sh.count[0] >> 16;
    sh.count[0] &= 0xffffu;
    if (sh.last == 0x8000u) sh.last = 0x7fffu;
    if (sh.last == 0x7fffu)
      sh.lowest += minus;
    else if (plus + minus < 65536u)
      sh.count[0x7fff] += minus;
    else
      sh.count[0x7fff] &= 0xffff0000u;  // too many: the sum will say so
    // all of the lowest together; its place in the table says that there is one
    const unsigned at = sh.last & 0x7fff, half = sh.last >> 15 << 4;
    sh.lowest += sh.count[at] >> half & 0xffffu;
    sh.count[at] = (sh.count[at] & ~(0xffffu << half)) | 1u << half;
  }
  __syncthreads();

  Extent e;
  e.hi = e.lo = logit_at<T>(first);
  e.at = 0;
  const RowScale r = row_scale(a, row, e);
  const u64 least = least_weight(a, row, r);
  // Sums of groups of 64 ranks. A list of those that hold something, of which
  // each wave takes its share: weights are most of the work. Where top-k cuts
  // the row, the groups behind its border are left out, so members are counted
  // first.
  constexpr int WAVES = ROW_THREADS / 64;
  const double k = param(a.top_k, row);
  const unsigned lowest_rank = sh.last, lowest_count = sh.lowest;
  unsigned all = 0;
  u64 minp = 0;
#pragma unroll
  for (int i = 0; i < 128 / WAVES; ++i) {
    const int b = i * WAVES + wave;  // 16 lanes read 64 words
    const i32x4 c = *reinterpret_cast<const i32x4*>(sh.count + b * 256 + lane * 4);
    const int group = b * 4 + lane / 16;
    if (r.by_k) {
      const u16x2 ones = {1, 1}, upper = {0, 1};
      unsigned both = 0, hi = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int word = c[j];
        const u16x2 n = __builtin_bit_cast(u16x2, word);
        both = __builtin_amdgcn_udot2(n, ones, both, false);
        hi = __builtin_amdgcn_udot2(n, upper, hi, false);
      }
      all += both;
      unsigned lo = both - hi;
      // NaN and -inf are no members
      const int first_word = b * 256 + lane * 4;
      if (b * 256 < (int)Ranks<T>::INF) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (first_word + j < (int)Ranks<T>::INF) lo -= (unsigned)c[j] & 0xffffu;
      }
      if (b * 256 >= (int)(Ranks<T>::NONE & 0x7f00u)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (first_word + j >= (int)(Ranks<T>::NONE & 0x7fffu)) hi -= (unsigned)c[j] >> 16;
      }
      lo = row_run_up(lo);
      hi = row_run_up(hi);
      if ((lane & 15) == 15) {
        sh.members[group] = lo;
        sh.members[group + GROUPS / 2] = hi;
      }
    } else {
      const unsigned some = row_or((unsigned)(c[0] | c[1] | c[2] | c[3]));
      if ((lane & 15) == 15 && some) {
        if (some & 0xffffu) sh.group_list[atomicAdd(&sh.groups, 1u)] = (unsigned short)group;
        if (some >> 16)
          sh.group_list[atomicAdd(&sh.groups, 1u)] = (unsigned short)(group + GROUPS / 2);
      }
    }
  }
  __syncthreads();
  if (r.by_k) {
    // in the table the lowest value is one
    if (t == 0) all += lowest_count - 1u;
    unsigned own = sh.members[t];
    if (t == (int)(lowest_rank >> 6) && lowest_rank >= Ranks<T>::INF &&
        lowest_rank < Ranks<T>::NONE)
      own += lowest_count - 1u;
    const unsigned through = block_run_up(own, sh.wave_members);
    sh.members[t] = through;  // thread t has group t
    const bool in = own && (double)(through - own) < k;
    const u64 who = __ballot(in);
    unsigned at = 0;
    if (lane == 0 && who) at = atomicAdd(&sh.groups, (unsigned)__popcll(who));
    at = __builtin_amdgcn_readfirstlane(at) +
         __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32),
                                   __builtin_amdgcn_mbcnt_lo((unsigned)who, 0u));
    if (in) sh.group_list[at] = (unsigned short)t;
    __syncthreads();
  }
  const int groups = (int)sh.groups, share = (groups + WAVES - 1) / WAVES;
  for (int i = wave * share; i < min(groups, wave * share + share); ++i) {
    const int group = __builtin_amdgcn_readfirstlane(sh.group_list[i]);
    const unsigned rank = (unsigned)group * 64 + lane;
    unsigned n = count_at(sh, rank);
    if (!r.by_k) all += n;
    if (rank < Ranks<T>::INF || rank >= Ranks<T>::NONE) n = 0;
    const u64 w = weight(r, logit_at<T>(rank));
    u64 mass = n * w;
    if (w >= least) minp += mass;
    mass = wave_run_up(mass);
    if (lane == 63) sh.mass[group] = mass;
  }
  all = wave_run_up(all);
  minp = wave_run_up(minp);
  if (lane == 63) {
    atomicAdd(&sh.logits, all);
    atomicAdd(&sh.minp, minp);
  }
  __syncthreads();
  if (sh.logits != (unsigned)a.vocab) {  // uniform: the row has to be kept whole
    __syncthreads();
    whole_row<T>(a, row, shared.row);
    return;
  }
  sh.mass[t] = block_run_up(sh.mass[t], sh.wave_mass);  // as of members
  __syncthreads();

  u64 kept = sh.mass[GROUPS - 1];
  if (r.by_k && k < (double)sh.members[GROUPS - 1]) {
    find_border<T>(sh, r, true, (u64)k);
    kept = sh.kept;
  }
  if (r.by_p) {
    find_border<T>(sh, r, false, share_of(param(a.top_p, row), kept));
    kept = sh.kept;
  }
  kept = min(kept, sh.minp);
  find_border<T>(sh, r, false, draw_border(param(a.u, row), kept));
  const unsigned rank = sh.rank;
  const unsigned copies = count_at(sh, rank);
  if (copies > MANY_COPIES) {
    const int token = index_of(sh, x, vocab, rank, sh.copy);
    if (t == 0) a.token[row] = token;
    return;
  }
  // A few copies: their indices to a list, from the last loads back to the
  // first; the answer has `copy` of them below it.
  const Wanted wanted(rank);
  auto list = [&](int at) {
    const unsigned i = atomicAdd(&sh.listed, 1u);
    if (i < MANY_COPIES) sh.list[i] = (unsigned)at;
  };
  if (edge < vocab && !wanted.differ((int)edge_bits)[0]) list(edge);
  if (v0 >= vecs) v0 -= STEP;  // a wave without vectors
  while (v0 >= 0) {
    i32x4 next[AHEAD];
    if (v0 >= STEP) load(next, v0 - STEP);
#pragma unroll
    for (int l = 0; l < AHEAD; ++l) {
      const int at = v0 + l * ROW_THREADS + lane;
      if (at >= vecs || !wanted.among(v[l])) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!wanted.differ(v[l][j / 2])[j % 2]) list(head + at * 8 + j);
    }
    v0 -= STEP;
#pragma unroll
    for (int l = 0; l < AHEAD; ++l) v[l] = next[l];
  }
  __syncthreads();
  if (wave != 0) return;
  const unsigned listed = min(sh.listed, MANY_COPIES);
  const unsigned own = sh.list[min((unsigned)lane, MANY_COPIES - 1)];
  unsigned below = 0;
  for (unsigned i = 0; i < listed; ++i) below += sh.list[i] < own;
  if ((unsigned)lane < listed && below == sh.copy) a.token[row] = own;
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  const dim3 rows((unsigned)a.rows), threads(ROW_THREADS);
  if constexpr (sizeof(T) == 2) {
    row_table_kernel<T><<<rows, threads, 0, stream>>>(a);
  } else if (a.chunks == 0) {
    row_whole_kernel<T><<<rows, threads, 0, stream>>>(a);
  } else {
    const dim3 grid((unsigned)a.chunks * (unsigned)a.rows);
    chunk_max_kernel<T><<<grid, dim3(CHUNK_THREADS), 0, stream>>>(a);
    if (a.binned) chunk_bins_kernel<T><<<grid, dim3(CHUNK_THREADS), 0, stream>>>(a);
    row_pick_kernel<T><<<rows, threads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_type(ActType t, const SampleArgs& a, hipStream_t stream) {
  switch (t) {
    case ActType::bf16: return launch<__bf16>(a, stream);
    case ActType::f16: return launch<_Float16>(a, stream);
    case ActType::f32: return launch<float>(a, stream);
  }
  return hipErrorInvalidValue;
}

// A setting's values from row `first` on.
SampleParam from_row(SampleParam p, long first) {
  const int size = p.kind == SampleParam::f32 || p.kind == SampleParam::i32 ? 4 : 8;
  if (p.kind != SampleParam::value_) p.ptr = static_cast<const char*>(p.ptr) + first * size;
  return p;
}

// Rows to a launch, whose threads are counted in 32 bits: a row takes 1024, or
// 256 a chunk, of which there are 2048 more than rows at most.
constexpr int MOST_ROWS = 1 << 21;

struct Plan {
  int chunk, chunks;
  size_t bins_at, scales_at, bytes;
};

Plan plan_of(ActType t, int rows, int vocab) {
  // At least 4096 logits a chunk; more where there are chunks enough for the
  // chip without that, so that fewer histograms are written.
  Plan p{};
  if (rows > MOST_ROWS) rows = MOST_ROWS;
  if (t != ActType::f32 || vocab <= (rows >= MANY ? WHOLE_MANY : WHOLE)) return p;
  const long want = ((long)rows * vocab + 2047) / 2048;
  p.chunk = want <= 4096 ? 4096 : (int)(((want < vocab ? want : vocab) + 511) / 512 * 512);
  p.chunks = (vocab + p.chunk - 1) / p.chunk;
  p.bins_at = ((size_t)rows * p.chunks * sizeof(ChunkMax) + 255) / 256 * 256;
  p.scales_at = p.bins_at + (size_t)rows * p.chunks * sizeof(ChunkBins);
  p.bytes = p.scales_at + (size_t)rows * sizeof(RowScale);
  return p;
}

}  // namespace

size_t sample_workspace(ActType t, int rows, int vocab) {
  return rows > 0 && vocab > 0 ? plan_of(t, rows, vocab).bytes : 0;
}

hipError_t sample(ActType t, const void* logits, long stride, int rows,
                  int vocab, SampleParam temperature, SampleParam top_k,
                  SampleParam top_p, SampleParam min_p, SampleParam u,
                  void* workspace, int64_t* token, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  if (vocab <= 0) return hipErrorInvalidValue;
  if (t != ActType::f32 && vocab > SAMPLE_MOST_16) return hipErrorInvalidValue;
  const Plan p = plan_of(t, rows, vocab);
  int shift = 45;  // sums of `vocab` weights stay below 2^62
  while (vocab > (int64_t(1) << (62 - shift))) --shift;
  char* const work = static_cast<char*>(workspace);
  const SampleArgs a{logits, stride, rows, vocab, p.chunk, p.chunks, shift,
                     temperature, top_k, top_p, min_p, u,
                     reinterpret_cast<ChunkMax*>(work),
                     reinterpret_cast<ChunkBins*>(work + p.bins_at),
                     reinterpret_cast<RowScale*>(work + p.scales_at),
                     temperature.kind != SampleParam::value_ || temperature.value > 0,
                     token};
  // one launch after the other, in the same workspace
  for (long first = 0; first < rows; first += MOST_ROWS) {
    SampleArgs now = a;
    now.logits = static_cast<const char*>(logits) + first * stride * (t == ActType::f32 ? 4 : 2);
    now.rows = (int)(rows - first < MOST_ROWS ? rows - first : MOST_ROWS);
    for (SampleParam* p : {&now.temperature, &now.top_k, &now.top_p, &now.min_p, &now.u})
      *p = from_row(*p, first);
    now.token = token + first;
    const hipError_t e = launch_type(t, now, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace lpx
