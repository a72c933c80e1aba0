// y[M, N] = a[m] w[n] sum over k of X[m, k] W[n, k] (+ bias[n]): a product of 8-bit integers with a float32 scale for every
// token and every output channel, and the kernel that makes the integers of a row: X[m, k] = round(x[m, k] / a[m]) within -127 .. 127,
// a[m] = max_k |x[m, k]| / 127, ties to even, float32 throughout.  The sums are exact in 32 bits up to a K of 133,144 (127^2 K <
// 2^31), so neither their order nor where K is cut shows in a result: y is rounded in the sum's conversion to float32 (beyond
// 2^24), twice by the scales, and once to its type.
//
// Few rows: every byte of W is read once, straight into the matrix instruction's operand, and the product is bound by that
// reading (one row by 6,144 x 6,144: 13.2 us, 37.7 MB, of which a launch and the latencies of two reads are 5).
// More rows: gemm_wide.h's loop.  Up to 64 rows it is bound by the reading of W (37 x 28,672 x 4,096: 21.8 us, 5.4 TB/s); 2,048 x
// 43,008 x 6,144 runs at 2.2 POP/s in 490 us, bound by LDS and matrix cores in turn: by count a step's operands are read in 0.43 us and
// multiplied in 0.43, and the step takes 0.85 (in bfloat16, with twice the products' time for as many bytes, the reads hide).
#include <type_traits>

#include "gemm_wide.h"

CWM_DEFINE_ERROR_API

#define INT8_MAX_K 131072

// ---- the integers of a row ---------------------------------------------------------------- //
template <typename T> __device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* p, float (&x)[4]) {
  const float4 v = *(const float4*)p;
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <> __device__ __forceinline__ void load4<bf16_t>(const bf16_t* p, float (&x)[4]) {
  const uint2 v = *(const uint2*)p;
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u), x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}

// A true quotient: ties are common among short numbers, and a product with 1 / a would decide them otherwise.  It ends at 127: a
// scale of one or two of float32's smallest steps (a row up to 2e-41 or so) is off by a large part of itself, and quotients would
// reach 190.
__device__ __forceinline__ int int8_of(float x, float a) { return (int)fminf(fmaxf(rintf(x / a), -127.f), 127.f); }

// The integers of N numbers.  A product with 1 / a decides one except next to a tie, where it may be off by its own rounding (the
// quotient is at most 127, a reciprocal off by 2^-23 and a product by 2^-24 make it 2.3e-5): there it is the quotient.  A scale with
// a reciprocal is 2^-128 at least, off by 2^-22 of itself at most, and its quotients round to 127 at most.
template <int N> __device__ __forceinline__ void int8_all(const float (&x)[N], float a, int (&c)[N]) {
  const float inv = __builtin_amdgcn_rcpf(a);  // an infinity for the smallest scales
  float r[N], off = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float t = x[e] * inv;
    r[e] = rintf(t);
    off = fmaxf(off, fabsf(t - r[e]));
  }
  if (off >= 0.4999f || inv == __builtin_inff()) {
#pragma unroll
    for (int e = 0; e < N; ++e) c[e] = int8_of(x[e], a);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) c[e] = (int)r[e];
  }
}
__device__ __forceinline__ uint32_t four_bytes(int a, int b, int c, int d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// One block a row: the largest magnitude, then the integers in a row of Kp.  Zeros fill it up, from K on, or (`shift`, Kp - K) ahead of
// the integers from the last multiple of 128 on, which then end with the row.  A row with a NaN or an infinity in it has a NaN
// for its scale (and zeros for its integers).
// PIECES > 0 (rows of whole pieces of eight, 16-byte aligned, up to 4,096 PIECES columns): a thread keeps that many pieces of eight
// in registers, all loaded at once: few rows are bound by that latency, many by the memory (8 rows of 21,504 5.0 us, number by number
// 20.9; 2,048 of 6,144 11.4).
#define ROW_THREADS 512
template <typename T, int PIECES>
__global__ void __launch_bounds__(ROW_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long x_stride, int8_t* __restrict__ codes, long c_stride, float* __restrict__ scale, int K, int Kp, int shift) {
  __shared__ float scratch[16];
  const T* row = x + (size_t)blockIdx.x * x_stride;
  int8_t* out = codes + (size_t)blockIdx.x * c_stride;
  const int tail = K / 128 * 128;  // from here on the integers move on by `shift`
  uint32_t top = 0;  // magnitudes as integers: an infinity and a NaN are larger than every number
  float v[PIECES > 0 ? PIECES : 1][8];
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = min(8 * (int)(threadIdx.x + ROW_THREADS * i), K - 8);  // past the row its last piece again
      float lo[4], hi[4];
      load4(row + k, lo), load4(row + k + 4, hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = lo[e], v[i][4 + e] = hi[e];
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
  } else {
    for (int k = threadIdx.x; k < K; k += ROW_THREADS) top = max(top, __float_as_uint(Elem<T>::load(row + k)) & 0x7fffffffu);
  }
  // the order of these floats is that of their bits; a NaN becomes an infinity
  const float most = block_max(top >= 0x7f800000u ? __builtin_inff() : __uint_as_float(top), scratch);
  const bool finite = most != __builtin_inff();
  const float a = most / 127.f;
  if (threadIdx.x == 0) scale[blockIdx.x] = finite ? a : __uint_as_float(0x7fc00000u);
  const bool none = !finite || a == 0.f;
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k = 8 * (threadIdx.x + ROW_THREADS * i);
      if (k >= K) break;
      int c[8] = {};
      if (!none) int8_all(v[i], a, c);
      *(uint2*)(out + k + (k >= tail ? shift : 0)) = make_uint2(four_bytes(c[0], c[1], c[2], c[3]), four_bytes(c[4], c[5], c[6], c[7]));
    }
    const int at = (shift > 0 ? tail : K) + 8 * threadIdx.x;
    if (8 * threadIdx.x < Kp - K) *(uint2*)(out + at) = make_uint2(0, 0);
  } else {
    for (int k = threadIdx.x; k < K; k += ROW_THREADS) out[k + (k >= tail ? shift : 0)] = none ? 0 : (int8_t)int8_of(Elem<T>::load(row + k), a);
    for (int i = threadIdx.x; i < Kp - K; i += ROW_THREADS) out[(shift > 0 ? tail : K) + i] = 0;
  }
}

static int quantize_rows(const void* x, long x_stride, int dtype, void* codes, long c_stride, float* scale, int M, int K, int Kp, int shift,
                         hipStream_t stream) {
  CWM_REQUIRE(M >= 0 && K > 0 && Kp >= K && c_stride >= Kp, "quantize_rows: bad sizes M=%d K=%d padded %d", M, K, Kp);
  if (M == 0) return 0;
  CWM_REQUIRE(x && codes && scale, "quantize_rows: a tensor is missing");
  const int size = dtype == CWM_BF16 ? 2 : 4;
  const bool whole = K % 8 == 0 && Kp % 8 == 0 && x_stride * size % 16 == 0 && c_stride % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)codes % 8 == 0;
  const int pieces = !whole || K > 64 * ROW_THREADS ? 0 : K <= 8 * ROW_THREADS ? 1 : K <= 16 * ROW_THREADS ? 2 : K <= 32 * ROW_THREADS ? 4 : 8;
  CWM_REQUIRE(shift == 0 || shift == Kp - K, "quantize_rows: integers move on to the end of their row or not at all");
#define QUANTIZE_ROWS(T, PIECES) \
  hipLaunchKernelGGL((quantize_rows_kernel<T, PIECES>), dim3(M), dim3(ROW_THREADS), 0, stream, (const T*)x, x_stride, (int8_t*)codes, c_stride, scale, K, Kp, shift)
#define QUANTIZE_PIECES(T)    \
  if (pieces == 0)            \
    QUANTIZE_ROWS(T, 0);      \
  else if (pieces == 1)       \
    QUANTIZE_ROWS(T, 1);      \
  else if (pieces == 2)       \
    QUANTIZE_ROWS(T, 2);      \
  else if (pieces == 4)       \
    QUANTIZE_ROWS(T, 4);      \
  else                        \
    QUANTIZE_ROWS(T, 8)
  if (dtype == CWM_BF16) {
    QUANTIZE_PIECES(bf16_t);
  } else {
    QUANTIZE_PIECES(float);
  }
  return cwm_launch_status("quantize_rows");
}

extern "C" int cwm_quantize_rows(const void* x, long x_stride, int dtype, void* codes, long c_stride, float* scale, int M, int K, int Kp,
                                 hipStream_t stream) {
  return quantize_rows(x, x_stride, dtype, codes, c_stride, scale, M, K, Kp, 0, stream);
}

// ---- few rows ------------------------------------------------------------------------------- //
// A block has 16 rows of W and up to 16 RT rows of X; its wavefronts take pieces of 128 columns in turn, lane 16 j + r the bytes
// 32 j .. 32 j + 31 of row r, which are two operands of the matrix instruction (the columns of a product may come in any order
// that both operands keep): a wavefront's load of W is 16 whole cache lines.  AHEAD pieces of a wavefront are in flight at a time,
// where K allows all of them: what the reading takes is then its latency once and the memory's rate.
// X comes from the caches, or (FUSED, up to FUSED_ROWS rows) every block makes the integers of x itself, in LDS, while its first
// pieces of W are under way: a second launch would cost more than the few thousand quotients.
#define FEW_WAVES 8
#define FUSED_ROWS 4
#define FUSED_SLOTS 8  // a thread's pieces of four values of x: eight of one row, four of each of two, two of each of four
#define FUSED_SLOT (4 * 64 * FEW_WAVES)

// FUSED: the number of rows of x that a block has room for (1, 2 or 4), or 0.
template <typename TX, typename T, int RT, int FUSED, int AHEAD>
__global__ void __launch_bounds__(64 * FEW_WAVES)
gemm_int8_few_kernel(const int8_t* __restrict__ X, long ldx, const float* __restrict__ a, const TX* __restrict__ x, long x_stride, bool x_aligned,
                     const int8_t* __restrict__ W, long ldw, const float* __restrict__ w_scale, const float* __restrict__ bias, T* __restrict__ y,
                     long ldy, int M, int N, int K, int rows_a_block) {
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];  // FUSED: [M][Kp]
  __shared__ __attribute__((aligned(16))) int4v sums[2][FEW_WAVES][RT][64];
  __shared__ float tops[FEW_WAVES][FUSED_ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, j = lane >> 4;
  const int m0 = blockIdx.y * 16 * RT;
  const int steps = (K + 127) / 128, Kp = 128 * steps;
  const int whole = K / 128;  // pieces that W holds whole
  const int rounds = (whole + FEW_WAVES * AHEAD - 1) / (FEW_WAVES * AHEAD);
  typedef const int4v* pieces;
  const int4v zero = (int4v){0, 0, 0, 0};
  int4v w[AHEAD][2];
  const int n_begin = blockIdx.x * rows_a_block, n_end = min(n_begin + rows_a_block, N);
  // lanes past the block's last row read that one again, which costs no memory
  auto row_of = [&](int n0) { return W + (size_t)min(n0 + r, n_end - 1) * ldw + 32 * j; };
  auto load_w = [&](int n0, int round) {  // no branch around a load: past the last piece that one again, which is not multiplied
    const int8_t* row = row_of(n0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[u][h] = __builtin_nontemporal_load((pieces)(row + 128 * min(wave + FEW_WAVES * (round * AHEAD + u), whole - 1) + 16 * h));
  };
  float scale_row[FUSED > 0 ? FUSED : 1];

  if constexpr (FUSED > 0) {
    // The rows of x, loaded ahead of W: loads return in order, so behind W's they would wait for the whole of it.
    constexpr int A_ROW = FUSED_SLOTS / FUSED;
    float v[FUSED_SLOTS][4];
#pragma unroll
    for (int i = 0; i < FUSED_SLOTS; ++i) {
      const int m = i / A_ROW, k = i % A_ROW * FUSED_SLOT + 4 * threadIdx.x;
      const bool have = m < M && k < K;  // K is a multiple of 16
      const TX* p = x + (have ? (size_t)m * x_stride + k : 0);
      if (x_aligned) {
        load4(p, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = Elem<TX>::load(p + (have ? e : 0));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = have ? v[i][e] : 0.f;
    }
    if (rounds > 0) load_w(n_begin, 0);
#pragma unroll
    for (int m = 0; m < FUSED; ++m) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < A_ROW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[m * A_ROW + i][e]) & 0x7fffffffu);
      const float most = wave_max(top >= 0x7f800000u ? __builtin_inff() : __uint_as_float(top));
      if (lane == 0) tops[wave][m] = most;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < FUSED; ++m) {
      float most = tops[0][m];
#pragma unroll
      for (int u = 1; u < FEW_WAVES; ++u) most = fmaxf(most, tops[u][m]);
      scale_row[m] = most == __builtin_inff() ? __uint_as_float(0x7fc00000u) : most / 127.f;
    }
#pragma unroll
    for (int i = 0; i < FUSED_SLOTS; ++i) {
      const int m = i / A_ROW, k = i % A_ROW * FUSED_SLOT + 4 * threadIdx.x;
      if (m >= M || k >= Kp) continue;
      int c[4] = {};
      if (scale_row[m] > 0.f) int8_all(v[i], scale_row[m], c);  // not of a row of zeros, nor where it is a NaN
      *(uint32_t*)(codes + (size_t)m * Kp + k) = four_bytes(c[0], c[1], c[2], c[3]);
    }
    __syncthreads();
  } else {
    if (rounds > 0) load_w(n_begin, 0);
  }

  const int8_t* x_row[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if constexpr (FUSED > 0)
      x_row[rt] = codes + (size_t)min(r, M - 1) * Kp + 32 * j;
    else
      x_row[rt] = X + (size_t)min(m0 + 16 * rt + r, M - 1) * ldx + 32 * j;
  }
  for (int n0 = n_begin, buffer = 0; n0 < n_end; n0 += 16, buffer ^= 1) {
    int4v acc[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[rt] = zero;
    for (int round = 0; round < rounds; ++round) {
      int4v xp[AHEAD][RT][2];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) xp[u][rt][h] = *(pieces)(x_row[rt] + 128 * min(wave + FEW_WAVES * (round * AHEAD + u), whole - 1) + 16 * h);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int4v wp = wave + FEW_WAVES * (round * AHEAD + u) < whole ? w[u][h] : zero;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wp, xp[u][rt][h], acc[rt], 0, 0, 0);
        }
      // the block's next loads are under way before its sums are joined
      const bool more = round + 1 < rounds;
      if (more || n0 + 16 < n_end) load_w(more ? n0 : n0 + 16, more ? round + 1 : 0);
    }
    // K's end: X holds zeros up to a multiple of 128, W ends at K, a multiple of 16
    if (whole < steps && wave == whole % FEW_WAVES) {
      const int8_t* row = row_of(n0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int4v wp = 128 * whole + 32 * j + 16 * h < K ? *(pieces)(row + 128 * whole + 16 * h) : zero;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wp, *(pieces)(x_row[rt] + 128 * whole + 16 * h), acc[rt], 0, 0, 0);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sums[buffer][wave][rt][lane] = acc[rt];
    __syncthreads();  // two buffers: what is written next is read two barriers on
    // lane 16 j + r holds the sums of row r of X and the columns 4 j .. 4 j + 3
    for (int rt = wave; rt < RT; rt += FEW_WAVES) {
      int4v sum = sums[buffer][0][rt][lane];
#pragma unroll
      for (int v = 1; v < FEW_WAVES; ++v) sum += sums[buffer][v][rt][lane];
      const int m = m0 + 16 * rt + r;
      if (m >= M) continue;
      float am = 0.f;
      if constexpr (FUSED > 0) {
#pragma unroll
        for (int u = 0; u < FUSED; ++u) am = r == u ? scale_row[u] : am;
      } else {
        am = a[m];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + 4 * j + e;
        if (n < n_end) Elem<T>::store(y + (size_t)m * ldy + n, (float)sum[e] * am * w_scale[n] + (bias ? bias[n] : 0.f));
      }
    }
  }
}

// ---- many rows --------------------------------------------------------------------------------- //
#define WIDE_BAND 8

struct Int8Order {
  int m_tiles, n_tiles, columns;  // of a tile: all that it has room for, or fewer
  __device__ __forceinline__ void place(int t, int& tm, int& tn) const {  // bands of WIDE_BAND row tiles, in a band column by column
    const int band = t / (WIDE_BAND * n_tiles), in_band = t - band * WIDE_BAND * n_tiles;
    const int rows = min(WIDE_BAND, m_tiles - band * WIDE_BAND);
    tn = in_band / rows;
    tm = band * WIDE_BAND + in_band - tn * rows;
  }
};

template <int WM, int WN>
struct Int8Source {
  const bf16_t *A, *W;
  long lda, ldw;  // in pairs of bytes
  int M, N, w_last, begin, steps, lane, wave;  // the steps of K from `begin` on
  Int8Order order;
  const bf16_t *a, *w;
  int first_step;
  uint32_t off[WideShape<WM, WN>::ND];
  static constexpr bool W_TILES = false;
  __device__ __forceinline__ const bf16_t* base(int p) const { return p < WideShape<WM, WN>::BM / 8 ? a : w; }
  __device__ __forceinline__ void enter(int tile) {
    constexpr int BM = WideShape<WM, WN>::BM, BN = WideShape<WM, WN>::BN;
    int tm, tn;
    order.place(tile, tm, tn);
    const int m0 = tm * BM, n0 = tn * order.columns, last = min(order.columns, N - n0) - 1;
    a = A + (size_t)m0 * lda;
    w = W + (size_t)n0 * ldw;
    first_step = tn % steps;
#pragma unroll
    for (int i = 0; i < WideShape<WM, WN>::ND; ++i) {
      const int p = min(wave + 8 * i, WideShape<WM, WN>::PIECES - 1);
      const int row = 8 * p + (lane >> 3);
      // rows past the matrix, or the tile's columns, read the last one: their sums are not stored
      if (p < BM / 8)
        off[i] = (uint32_t)(((size_t)min(row, M - 1 - m0) * lda + 8 * ((lane & 7) ^ ((row >> 1) & 7))) * 2);
      else
        off[i] = (uint32_t)(((size_t)min(row - BM, last) * ldw + 8 * ((lane & 7) ^ wide_w_key<WN>(row - BM))) * 2);
    }
  }
};

template <int WM, int WN, typename T>
struct Int8Sink {
  T* C;
  long ldc;
  const float *a, *w_scale, *bias;
  int M, N, lane, wave;
  Int8Order order;
  static constexpr int STORES = sizeof(T) == 4 ? WM * WN : WM * WN / 2;

  __device__ __forceinline__ bool store(int tile, int4v (&acc)[WM][WN]) const {
    constexpr int BM = WideShape<WM, WN>::BM, BN = WideShape<WM, WN>::BN;
    int tm, tn;
    order.place(tile, tm, tn);
    const int r = lane & 15, j = lane >> 4, wm = wave >> 2, wn = wave & 3;
    const int m0 = tm * BM + wm * WM * 16 + r;
    const int n0 = tn * order.columns + wn * WN * 16 + 4 * WN * j, end = min(N, (tn + 1) * order.columns);
    if constexpr (std::is_same<T, int>::value) {  // sums of a part of K: rows of whole tiles
#pragma unroll
      for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int b = 0; b < WN; ++b)
          if (m0 + 16 * i < M) *(int4v*)(C + (size_t)(m0 + 16 * i) * ldc + n0 + 4 * b) = acc[i][b];
      return false;
    } else {
      float am[WM], ws[WN][4], bs[WN][4];
#pragma unroll
      for (int i = 0; i < WM; ++i) am[i] = a[min(m0 + 16 * i, M - 1)];
#pragma unroll
      for (int b = 0; b < WN; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = min(n0 + 4 * b + e, N - 1);
          ws[b][e] = w_scale[n];
          bs[b][e] = bias ? bias[n] : 0.f;
        }
      // Waited for here, by an instruction that the compiler knows of: loads that it takes to be under way at the loop's head
      // make it wait for all of the loop's own loads in every step (2,048 x 43,008 x 6,144 663 us, 1.24 us a step).
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      const bool full = (tm + 1) * BM <= M && tn * order.columns + BN <= end;
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        const int m = m0 + 16 * i;
        if (m >= M) continue;
        T* row = C + (size_t)m * ldc + n0;
        float v[WN][4];
#pragma unroll
        for (int b = 0; b < WN; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[b][e] = (float)acc[i][b][e] * am[i] * ws[b][e] + bs[b][e];
#pragma unroll
        for (int b = 0; b < WN; b += 2) {
          if (n0 + 4 * b + 7 < end) {  // a row may begin anywhere: 16 bytes to any address
            if constexpr (sizeof(T) == 4) {
              __builtin_memcpy(row + 4 * b, v[b], 16);
              __builtin_memcpy(row + 4 * b + 4, v[b + 1], 16);
            } else {
              const uint4 w = make_uint4(pack2_bf16(v[b][0], v[b][1]), pack2_bf16(v[b][2], v[b][3]), pack2_bf16(v[b + 1][0], v[b + 1][1]),
                                         pack2_bf16(v[b + 1][2], v[b + 1][3]));
              __builtin_memcpy(row + 4 * b, &w, 16);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n0 + 4 * b + e < end) Elem<T>::store(row + 4 * b + e, v[b + e / 4][e % 4]);
          }
        }
      }
      return full;
    }
  }
};

// T int: the sums of `parts` parts of K are written to y, [parts][M][ldy], a block a tile of one part.
template <int WM, int WN, typename T, bool ONCE>
__global__ void __launch_bounds__(512, 2)
gemm_int8_wide_kernel(const int8_t* __restrict__ X, long ldx, const float* __restrict__ a, const int8_t* __restrict__ W, long ldw,
                      const float* __restrict__ w_scale, const float* __restrict__ bias, T* __restrict__ y, long ldy, int M, int N,
                      int K, int m_tiles, int n_tiles, int columns, int parts) {
  typedef WideShape<WM, WN> Shape;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Shape::S * Shape::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the XCDs (block number modulo 8) take consecutive runs of tiles, their blocks in turn
  const int tiles = m_tiles * n_tiles, total = tiles * parts, groups = min(8, (int)gridDim.x);
  const int xcd = blockIdx.x % groups, idx = blockIdx.x / groups;
  const int blocks = ((int)gridDim.x + groups - 1 - xcd) / groups;
  const int per = total / groups, rest = total % groups;
  const int first = xcd * per + min(xcd, rest), count = per + (xcd < rest ? 1 : 0);
  const int mine = (count - idx + blocks - 1) / blocks;
  const Int8Order order = {m_tiles, n_tiles, columns};
  constexpr bool PARTS = std::is_same<T, int>::value;
  const int all = (K + 127) / 128, part = PARTS ? (first + idx) / tiles : 0;
  const int begin = PARTS ? part * all / parts : 0, steps = PARTS ? (part + 1) * all / parts - begin : all;
  Int8Source<WM, WN> src = {(const bf16_t*)X, (const bf16_t*)W, ldx / 2, ldw / 2, M, N, (K - 128) / 2, begin, steps, lane, wave, order};
  Int8Sink<WM, WN, T> sink = {y + (size_t)part * M * ldy, ldy, a, w_scale, bias, M, N, lane, wave, order};
  wide_loop<WM, WN, Int8Sink<WM, WN, T>::STORES, WideInt8<ONCE, PARTS>>(lds, src, sink, first + idx - part * tiles, blocks, mine, steps);
}

// The columns of a tile where there is one tile of rows, and the reading of W is what counts: as many as give every compute unit the
// same number of them (37 x 28,672 x 4,096: 224 tiles of 128 columns on 256 units 23.3 us, 256 of 112 21.8; 8 x 43,008 x 6,144 52 and 45.5).
static int int8_columns(long N, int most, long tiles, int units) {
  const long rounds = (tiles + units - 1) / units, columns = (N + rounds * units - 1) / (rounds * units);
  return (int)(columns > most ? most : (columns + 7) / 8 * 8);
}

// The parts' sums, [parts][M][ldp], added, scaled and rounded.  A thread has four columns of a row.
template <typename T>
__global__ void __launch_bounds__(256)
gemm_int8_join_kernel(const int* __restrict__ sums, long ldp, int parts, const float* __restrict__ a, const float* __restrict__ w_scale,
                      const float* __restrict__ bias, T* __restrict__ y, long ldy, int M, int N) {
  const int n = 4 * (blockIdx.x * 256 + threadIdx.x), m = blockIdx.y;
  if (n >= N) return;
  int4v sum = *(const int4v*)(sums + (size_t)m * ldp + n);
  for (int p = 1; p < parts; ++p) sum += *(const int4v*)(sums + ((size_t)p * M + m) * ldp + n);
  const float am = a[m];
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = min(n + e, N - 1);
    const float ws = w_scale[at], bs = bias ? bias[at] : 0.f;
    v[e] = (float)sum[e] * am * ws + bs;
  }
  T* row = y + (size_t)m * ldy + n;
  if (n + 3 < N) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(row, v, 16);
    } else {
      const uint2 w = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
      __builtin_memcpy(row, &w, 8);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) Elem<T>::store(row + e, v[e]);
  }
}

// y = x W^T (+ bias): x [M][x_stride] of x_dtype; W int8 [N][ldw] with its float32 scales [N]; y of y_dtype.  `codes`, `a`: room
// for the integers of x, [M][K rounded up to 128] bytes, and their scales, M floats (neither with tile -1).
// `tile`: -1 few rows whose integers every block makes itself (M <= 4); 0 few rows; 1 to 4 the tiles of many rows (256 x 128,
// 128 x 256, 64 x 128, 128 x 128), which need a K of 128 at least.  `parts` > 1 (tiles 3 and 4): K in that many parts, whose sums go to
// `sums`, [parts][M][N rounded up to 128] 32-bit integers, and are joined by a last launch.
extern "C" int cwm_linear_int8(const void* x, long x_stride, int x_dtype, void* codes, float* a, const void* W, long ldw, const float* w_scale,
                               const float* bias, void* y, int dtype, long ldy, int M, int N, int K, int units, int tile, int parts, int* sums,
                               hipStream_t stream) {
  CWM_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 16 == 0 && K <= INT8_MAX_K && units > 0, "linear_int8: bad sizes M=%d N=%d K=%d units=%d", M, N, K, units);
  if (M == 0) return 0;
  CWM_REQUIRE(x && W && w_scale && y, "linear_int8: a tensor is missing");
  CWM_REQUIRE(ldw % 16 == 0 && (uintptr_t)W % 16 == 0, "linear_int8: the weight's rows must be 16-byte aligned");
  CWM_REQUIRE(ldw >= K && ldy >= N, "linear_int8: row strides shorter than rows");
  const int x_size = x_dtype == CWM_BF16 ? 2 : 4, Kp = (K + 127) / 128 * 128;
  CWM_REQUIRE(parts >= 1 && parts <= Kp / 128 && (parts == 1 || ((tile == 3 || tile == 4) && sums && (uintptr_t)sums % 16 == 0)),
              "linear_int8: K in %d parts with tile %d", parts, tile);
  // Pieces of W that a wavefront of few rows has in flight at a time.  A round loads that many whether K has them or not, so of four and
  // six it takes what loads fewer in all, and six where that is equal (us with four and with six: one row by 6,144 columns of 6,144
  // 14.2 and 13.4, of 8,192 14.3 and 17.8; by 4,096 of 7,168 11.5 and 13.8, of 9,216 14.8 and 14.3, of 12,288 15.1 and 15.0, of 16,384
  // 18.4 and 19.3; eight rows by 4,096 of 16,384 28.3 and 30.6).
  const int a_wave = (K / 128 + FEW_WAVES - 1) / FEW_WAVES;  // pieces of a wavefront in all
  const int ahead = a_wave <= 2 ? 2 : (a_wave + 3) / 4 * 4 < (a_wave + 5) / 6 * 6 ? 4 : 6;
  // Two blocks a compute unit stay, each with the same number of rows of W: what one unit can have in flight is limited, so with
  // tiles dealt out one by one the units that get one more take that much longer (one row by 6,144 of 6,144: 384 tiles 14.6 us,
  // 512 blocks of 12 rows 13.2).
  const int few_rows = (N + 2 * units - 1) / (2 * units) > 4 ? (N + 2 * units - 1) / (2 * units) : 4, few_blocks = (N + few_rows - 1) / few_rows;
  if (tile == -1) {
    const int rows = M <= 2 ? M : 4;
    CWM_REQUIRE(M <= FUSED_ROWS && K <= FUSED_SLOTS / rows * FUSED_SLOT, "linear_int8: %d rows of %d columns are too many for one launch", M, K);
    const bool x_aligned = x_stride % 4 == 0 && (uintptr_t)x % (4 * x_size) == 0;
#define INT8_FUSED_RUN(TX, T, ROWS, AHEAD)                                                                                                       \
  hipLaunchKernelGGL((gemm_int8_few_kernel<TX, T, 1, ROWS, AHEAD>), dim3(few_blocks), dim3(64 * FEW_WAVES), M * Kp, stream, (const int8_t*)nullptr, \
                     0l, (const float*)nullptr, (const TX*)x, x_stride, x_aligned, (const int8_t*)W, ldw, w_scale, bias, (T*)y, ldy, M, N, K, few_rows)
#define INT8_FUSED_AHEAD(TX, T, ROWS)     \
  {                                       \
    if (ahead == 2)                       \
      INT8_FUSED_RUN(TX, T, ROWS, 2);     \
    else if (ahead == 4)                  \
      INT8_FUSED_RUN(TX, T, ROWS, 4);     \
    else                                  \
      INT8_FUSED_RUN(TX, T, ROWS, 6);     \
  }
#define INT8_FUSED(TX, T)             \
  {                                   \
    if (rows == 1)                    \
      INT8_FUSED_AHEAD(TX, T, 1)      \
    else if (rows == 2)               \
      INT8_FUSED_AHEAD(TX, T, 2)      \
    else                              \
      INT8_FUSED_AHEAD(TX, T, 4)      \
  }
    if (x_dtype == CWM_BF16 && dtype == CWM_BF16)
      INT8_FUSED(bf16_t, bf16_t)
    else if (x_dtype == CWM_BF16)
      INT8_FUSED(bf16_t, float)
    else if (dtype == CWM_BF16)
      INT8_FUSED(float, bf16_t)
    else
      INT8_FUSED(float, float)
    return cwm_launch_status("linear_int8 (one launch)");
  }
  CWM_REQUIRE(codes && a && (uintptr_t)codes % 16 == 0, "linear_int8: room for the integers is missing");
  const int shift = tile > 0 ? Kp - K : 0;
  if (int status = quantize_rows(x, x_stride, x_dtype, codes, Kp, a, M, K, Kp, shift, stream)) return status;
  const int8_t* X = (const int8_t*)codes;
  const long ldx = Kp;
  if (tile == 0) {
    const int row_tiles = (M + 15) / 16, rt = row_tiles > 1 ? 4 : 1;  // more than one for a K below a tile's
    CWM_REQUIRE((row_tiles + rt - 1) / rt <= 65535, "linear_int8: too many rows");
    const dim3 grid(few_blocks, (row_tiles + rt - 1) / rt);
#define INT8_FEW(T, RT, AHEAD)                                                                                                                       \
  hipLaunchKernelGGL((gemm_int8_few_kernel<float, T, RT, 0, AHEAD>), grid, dim3(64 * FEW_WAVES), 0, stream, X, ldx, a, (const float*)nullptr, 0l, \
                     false, (const int8_t*)W, ldw, w_scale, bias, (T*)y, ldy, M, N, K, few_rows)
#define INT8_FEW_ROWS(T)               \
  if (rt == 4)                         \
    INT8_FEW(T, 4, 2);                 \
  else if (ahead == 2)                 \
    INT8_FEW(T, 1, 2);                 \
  else if (ahead == 4)                 \
    INT8_FEW(T, 1, 4);                 \
  else                                 \
    INT8_FEW(T, 1, 6)
    if (dtype == CWM_BF16) {
      INT8_FEW_ROWS(bf16_t);
    } else {
      INT8_FEW_ROWS(float);
    }
    return cwm_launch_status("linear_int8 (few rows)");
  }
  CWM_REQUIRE(K >= 128, "linear_int8: the tiles of many rows take a K of 128 and more, not %d", K);
  CWM_REQUIRE(ldx < (1L << 23) && ldw < (1L << 23), "linear_int8: row strides too long for 32-bit offsets");
  CWM_REQUIRE(tile >= 1 && tile <= 4, "linear_int8: no tile %d", tile);
  if (parts > 1) {
    const long m_tiles = tile == 3 ? (M + 63) / 64 : (M + 127) / 128, n_tiles = (N + 127) / 128, ldp = n_tiles * 128;
    CWM_REQUIRE(m_tiles * n_tiles * parts <= 65536 && M <= 65535, "linear_int8: too many tiles to take K in parts");
    const dim3 grid((unsigned)(m_tiles * n_tiles * parts));
#define INT8_PARTS_RUN(WM, ONCE)                                                                                                              \
  hipLaunchKernelGGL((gemm_int8_wide_kernel<WM, 2, int, ONCE>), grid, dim3(512), 0, stream, (const int8_t*)X, ldx, a, (const int8_t*)W, ldw, \
                     w_scale, bias, sums, ldp, M, N, K, (int)m_tiles, (int)n_tiles, 128, parts)
    if (tile == 3 && m_tiles == 1)
      INT8_PARTS_RUN(2, true);
    else if (tile == 3)
      INT8_PARTS_RUN(2, false);
    else if (m_tiles == 1)
      INT8_PARTS_RUN(4, true);
    else
      INT8_PARTS_RUN(4, false);
    if (int status = cwm_launch_status("linear_int8 (K in parts)")) return status;
    const dim3 join((unsigned)((N + 1023) / 1024), (unsigned)M);
    if (dtype == CWM_BF16)
      hipLaunchKernelGGL((gemm_int8_join_kernel<bf16_t>), join, dim3(256), 0, stream, sums, ldp, parts, a, w_scale, bias, (bf16_t*)y, ldy, M, N);
    else
      hipLaunchKernelGGL((gemm_int8_join_kernel<float>), join, dim3(256), 0, stream, sums, ldp, parts, a, w_scale, bias, (float*)y, ldy, M, N);
    return cwm_launch_status("linear_int8 (joining parts)");
  }
#define INT8_WIDE_RUN(WM, WN, T, ONCE)                                                                                                      \
  hipLaunchKernelGGL((gemm_int8_wide_kernel<WM, WN, T, ONCE>), grid, dim3(512), 0, stream, (const int8_t*)X, ldx, a, (const int8_t*)W, ldw,  \
                     w_scale, bias, (T*)y, ldy, M, N, K, (int)m_tiles, (int)n_tiles, columns, 1)
#define INT8_WIDE(WM, WN)                                                                                          \
  {                                                                                                                \
    const long m_tiles = (M + 32 * WM - 1) / (32 * WM), all = (N + 64 * WN - 1) / (64 * WN);                       \
    const int columns = m_tiles > 1 ? 64 * WN : int8_columns(N, 64 * WN, all, units);                              \
    const long n_tiles = (N + columns - 1) / columns;                                                              \
    CWM_REQUIRE(m_tiles * n_tiles * (Kp / 128) < (1L << 31), "linear_int8: too many steps of tiles");                 \
    const dim3 grid((unsigned)(m_tiles * n_tiles < units ? m_tiles * n_tiles : units));                            \
    if (dtype == CWM_BF16 && m_tiles == 1)                                                                         \
      INT8_WIDE_RUN(WM, WN, bf16_t, true);                                                                         \
    else if (dtype == CWM_BF16)                                                                                    \
      INT8_WIDE_RUN(WM, WN, bf16_t, false);                                                                        \
    else if (m_tiles == 1)                                                                                         \
      INT8_WIDE_RUN(WM, WN, float, true);                                                                          \
    else                                                                                                           \
      INT8_WIDE_RUN(WM, WN, float, false);                                                                         \
  }
  if (tile == 1) INT8_WIDE(8, 2)
  if (tile == 2) INT8_WIDE(4, 4)
  if (tile == 3) INT8_WIDE(2, 2)
  if (tile == 4) INT8_WIDE(4, 2)
  return cwm_launch_status("linear_int8 (many rows)");
}
