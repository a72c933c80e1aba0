// y[M, N] = a[m] w[n] sum over k of X[m, k] W[n, k] (+ bias[n]): a product of 8-bit integers with a float32 scale for every
// token and every output channel, and the kernel that makes the integers of a row: X[m, k] = round(x[m, k] / a[m]),
// a[m] = max_k |x[m, k]| / 127, ties to even, float32 throughout.  The sums are exact in 32 bits up to a K of 133,144 (127^2 K <
// 2^31), so neither their order nor where K is cut shows in a result: y is rounded in the sum's conversion to float32 (beyond
// 2^24), twice by the scales, and once to its type.
//
// Few rows: every byte of W is read once, straight into the matrix instruction's operand, and the product is bound by that
// reading.  More rows: gemm_wide.h's loop.
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

__device__ __forceinline__ int int8_of(float x, float a) {
  return (int)rintf(x / a);  // a true quotient: ties are common among short numbers, and a product with 1 / a would decide them otherwise
}

// One block a row: the largest magnitude, then the integers, zeros from K to Kp.  A row with a NaN or an infinity in it has a
// NaN for its scale (and zeros for its integers).
template <typename T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, long x_stride, int8_t* __restrict__ codes, long c_stride, float* __restrict__ scale, int K, int Kp,
                     bool aligned) {
  __shared__ float scratch[16];
  const T* row = x + (size_t)blockIdx.x * x_stride;
  int8_t* out = codes + (size_t)blockIdx.x * c_stride;
  uint32_t top = 0;  // magnitudes as integers: an infinity and a NaN are larger than every number
  if (aligned) {
    for (int k = 4 * threadIdx.x; k < K; k += 1024) {
      float v[4];
      load4(row + k, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
  } else {
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(Elem<T>::load(row + k)) & 0x7fffffffu);
  }
  // the order of these floats is that of their bits; a NaN becomes an infinity
  const float most = block_max(top >= 0x7f800000u ? __builtin_inff() : __uint_as_float(top), scratch);
  const bool finite = most != __builtin_inff();
  const float a = most / 127.f;
  if (threadIdx.x == 0) scale[blockIdx.x] = finite ? a : __uint_as_float(0x7fc00000u);
  const bool none = !finite || a == 0.f;
  if (aligned) {
    for (int k = 4 * threadIdx.x; k < Kp; k += 1024) {
      uint32_t w = 0;
      if (k < K && !none) {
        float v[4];
        load4(row + k, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= ((uint32_t)int8_of(v[e], a) & 255u) << (8 * e);
      }
      *(uint32_t*)(out + k) = w;
    }
  } else {
    for (int k = threadIdx.x; k < Kp; k += 256) out[k] = k < K && !none ? (int8_t)int8_of(Elem<T>::load(row + k), a) : 0;
  }
}

extern "C" int cwm_quantize_rows(const void* x, long x_stride, int dtype, void* codes, long c_stride, float* scale, int M, int K, int Kp,
                                 hipStream_t stream) {
  CWM_REQUIRE(M >= 0 && K > 0 && Kp >= K && c_stride >= Kp, "quantize_rows: bad sizes M=%d K=%d padded %d", M, K, Kp);
  if (M == 0) return 0;
  CWM_REQUIRE(x && codes && scale, "quantize_rows: a tensor is missing");
  const int size = dtype == CWM_BF16 ? 2 : 4;
  const bool aligned = K % 4 == 0 && Kp % 4 == 0 && x_stride % 4 == 0 && c_stride % 4 == 0 && (uintptr_t)x % (4 * size) == 0 && (uintptr_t)codes % 4 == 0;
  if (dtype == CWM_BF16)
    hipLaunchKernelGGL(quantize_rows_kernel<bf16_t>, dim3(M), dim3(256), 0, stream, (const bf16_t*)x, x_stride, (int8_t*)codes, c_stride, scale, K, Kp, aligned);
  else
    hipLaunchKernelGGL(quantize_rows_kernel<float>, dim3(M), dim3(256), 0, stream, (const float*)x, x_stride, (int8_t*)codes, c_stride, scale, K, Kp, aligned);
  return cwm_launch_status("quantize_rows");
}

// ---- few rows ------------------------------------------------------------------------------- //
// A block has 16 rows of W and up to 16 RT rows of X; its wavefronts take pieces of 128 columns in turn, lane 16 j + r the bytes
// 32 j .. 32 j + 31 of row r, which are two operands of the matrix instruction (the columns of a product may come in any order
// that both operands keep): a wavefront's load of W is 16 whole cache lines.  X is read from the caches.
#define FEW_WAVES 4

template <typename T, int RT>
__global__ void __launch_bounds__(64 * FEW_WAVES)
gemm_int8_few_kernel(const int8_t* __restrict__ X, long ldx, const float* __restrict__ a, const int8_t* __restrict__ W, long ldw,
                     const float* __restrict__ w_scale, const float* __restrict__ bias, T* __restrict__ y, long ldy, int M, int N, int K) {
  __shared__ __attribute__((aligned(16))) int4v sums[FEW_WAVES][RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, j = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * RT;
  const int8_t* w_row = W + (size_t)min(n0 + r, N - 1) * ldw + 32 * j;
  const int8_t* x_row[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) x_row[rt] = X + (size_t)min(m0 + 16 * rt + r, M - 1) * ldx + 32 * j;
  int4v acc[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt] = (int4v){0, 0, 0, 0};
  const int4v none = (int4v){0, 0, 0, 0};
  // X holds zeros from K to the next multiple of 128, W ends at K: a piece of 16 columns lies before or past it as a whole
  auto piece = [&](int k, int4v (&w)[2], int4v (&x)[RT][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = k + 32 * j + 16 * h < K ? __builtin_nontemporal_load((const int4v*)(w_row + k + 16 * h)) : none;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) x[rt][h] = *(const int4v*)(x_row[rt] + k + 16 * h);
    }
  };
  const int steps = (K + 127) / 128;
#pragma unroll 4
  for (int s = wave; s < steps; s += FEW_WAVES) {
    int4v w[2], x[RT][2];
    piece(128 * s, w, x);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h], x[rt][h], acc[rt], 0, 0, 0);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) sums[wave][rt][lane] = acc[rt];
  __syncthreads();
  // lane 16 j + r holds the sums of row r of X and the columns 4 j .. 4 j + 3
  for (int rt = wave; rt < RT; rt += FEW_WAVES) {
    int4v sum = sums[0][rt][lane];
#pragma unroll
    for (int v = 1; v < FEW_WAVES; ++v) sum += sums[v][rt][lane];
    const int m = m0 + 16 * rt + r;
    if (m >= M) continue;
    const float am = a[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * j + e;
      if (n < N) Elem<T>::store(y + (size_t)m * ldy + n, (float)sum[e] * am * w_scale[n] + (bias ? bias[n] : 0.f));
    }
  }
}

// ---- many rows --------------------------------------------------------------------------------- //
#define WIDE_BAND 8

struct Int8Order {
  int m_tiles, n_tiles;
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
  int M, N, lane, wave;
  Int8Order order;
  const bf16_t *a, *w;
  uint32_t off[WideShape<WM, WN>::ND];
  static constexpr bool W_TILES = false;
  __device__ __forceinline__ const bf16_t* base(int p) const { return p < WideShape<WM, WN>::BM / 8 ? a : w; }
  __device__ __forceinline__ void enter(int tile) {
    constexpr int BM = WideShape<WM, WN>::BM, BN = WideShape<WM, WN>::BN;
    int tm, tn;
    order.place(tile, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    a = A + (size_t)m0 * lda;
    w = W + (size_t)n0 * ldw;
#pragma unroll
    for (int i = 0; i < WideShape<WM, WN>::ND; ++i) {
      const int p = min(wave + 8 * i, WideShape<WM, WN>::PIECES - 1);
      const int row = 8 * p + (lane >> 3);
      // rows past the matrix read its last one: their sums are not stored
      if (p < BM / 8)
        off[i] = (uint32_t)(((size_t)min(row, M - 1 - m0) * lda + 8 * ((lane & 7) ^ ((row >> 1) & 7))) * 2);
      else
        off[i] = (uint32_t)(((size_t)min(row - BM, N - 1 - n0) * ldw + 8 * ((lane & 7) ^ wide_w_key<WN>(row - BM))) * 2);
    }
  }
};

template <int WM, int WN, typename T>
struct Int8Sink {
  T* C;
  long ldc;
  const float *a, *w_scale, *bias;
  int M, N, lane, wave;
  bool vector;
  Int8Order order;
  static constexpr int STORES = 0;  // its loads and stores are waited for before the next tile's are counted

  __device__ __forceinline__ bool store(int tile, int4v (&acc)[WM][WN]) const {
    constexpr int BM = WideShape<WM, WN>::BM, BN = WideShape<WM, WN>::BN;
    int tm, tn;
    order.place(tile, tm, tn);
    const int r = lane & 15, j = lane >> 4, wm = wave >> 2, wn = wave & 3;
    const int m0 = tm * BM + wm * WM * 16 + r;
    const int n0 = tn * BN + wn * WN * 16 + 4 * WN * j;
    float ws[WN][4], bs[WN][4];
#pragma unroll
    for (int b = 0; b < WN; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = min(n0 + 4 * b + e, N - 1);
        ws[b][e] = w_scale[n];
        bs[b][e] = bias ? bias[n] : 0.f;
      }
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const int m = m0 + 16 * i;
      if (m >= M) continue;
      const float am = a[m];
      T* row = C + (size_t)m * ldc + n0;
#pragma unroll
      for (int b = 0; b < WN; ++b) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][b][e] * am * ws[b][e] + bs[b][e];
        if (vector && n0 + 4 * b + 3 < N) {
          if constexpr (sizeof(T) == 4)
            *(float4*)(row + 4 * b) = make_float4(v[0], v[1], v[2], v[3]);
          else
            *(uint2*)(row + 4 * b) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + 4 * b + e < N) Elem<T>::store(row + 4 * b + e, v[e]);
        }
      }
    }
    return false;
  }
};

template <int WM, int WN, typename T>
__global__ void __launch_bounds__(512, 2)
gemm_int8_wide_kernel(const int8_t* __restrict__ X, long ldx, const float* __restrict__ a, const int8_t* __restrict__ W, long ldw,
                      const float* __restrict__ w_scale, const float* __restrict__ bias, T* __restrict__ y, long ldy, bool vector, int M, int N,
                      int steps, int m_tiles, int n_tiles) {
  typedef WideShape<WM, WN> Shape;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Shape::S * Shape::STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the XCDs (block number modulo 8) take consecutive runs of tiles, their blocks in turn
  const int total = m_tiles * n_tiles, groups = min(8, (int)gridDim.x);
  const int xcd = blockIdx.x % groups, idx = blockIdx.x / groups;
  const int blocks = ((int)gridDim.x + groups - 1 - xcd) / groups;
  const int per = total / groups, rest = total % groups;
  const int first = xcd * per + min(xcd, rest), count = per + (xcd < rest ? 1 : 0);
  const int mine = (count - idx + blocks - 1) / blocks;
  const Int8Order order = {m_tiles, n_tiles};
  Int8Source<WM, WN> src = {(const bf16_t*)X, (const bf16_t*)W, ldx / 2, ldw / 2, M, N, lane, wave, order};
  Int8Sink<WM, WN, T> sink = {y, ldy, a, w_scale, bias, M, N, lane, wave, vector, order};
  wide_loop<WM, WN, Int8Sink<WM, WN, T>::STORES, WideInt8>(lds, src, sink, first + idx, blocks, mine, steps);
}

// X [M][ldx] int8 with zeros from K to the next multiple of 128 within ldx, a float32 [M]; W [N][ldw] int8; y of `dtype`.
// `tile`: 0 few rows; 1 to 4 the tiles of many rows (256 x 128, 128 x 256, 64 x 128, 128 x 128), which need K % 128 == 0.
extern "C" int cwm_gemm_int8(const void* X, long ldx, const float* a, const void* W, long ldw, const float* w_scale, const float* bias, void* y,
                             int dtype, long ldy, int M, int N, int K, int units, int tile, hipStream_t stream) {
  CWM_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 16 == 0 && K <= INT8_MAX_K && units > 0, "gemm_int8: bad sizes M=%d N=%d K=%d units=%d", M, N, K, units);
  if (M == 0) return 0;
  CWM_REQUIRE(X && a && W && w_scale && y, "gemm_int8: a tensor is missing");
  CWM_REQUIRE(ldx % 16 == 0 && ldw % 16 == 0 && (uintptr_t)X % 16 == 0 && (uintptr_t)W % 16 == 0, "gemm_int8: rows must be 16-byte aligned");
  CWM_REQUIRE(ldx >= (K + 127) / 128 * 128 && ldw >= K && ldy >= N, "gemm_int8: row strides shorter than rows");
  if (tile == 0) {
    const int row_tiles = (M + 15) / 16, rt = row_tiles >= 4 ? 4 : row_tiles >= 2 ? 2 : 1;
    CWM_REQUIRE((row_tiles + rt - 1) / rt <= 65535, "gemm_int8: too many rows");
    const dim3 grid((N + 15) / 16, (row_tiles + rt - 1) / rt);
#define INT8_FEW(T, RT)                                                                                                                       \
  hipLaunchKernelGGL((gemm_int8_few_kernel<T, RT>), grid, dim3(64 * FEW_WAVES), 0, stream, (const int8_t*)X, ldx, a, (const int8_t*)W, ldw,    \
                     w_scale, bias, (T*)y, ldy, M, N, K)
#define INT8_FEW_ROWS(T) \
  if (rt == 4)           \
    INT8_FEW(T, 4);      \
  else if (rt == 2)      \
    INT8_FEW(T, 2);      \
  else                   \
    INT8_FEW(T, 1)
    if (dtype == CWM_BF16) {
      INT8_FEW_ROWS(bf16_t);
    } else {
      INT8_FEW_ROWS(float);
    }
    return cwm_launch_status("gemm_int8 (few rows)");
  }
  CWM_REQUIRE(K % 128 == 0, "gemm_int8: the tiles of many rows take a K of a multiple of 128, not %d", K);
  CWM_REQUIRE(ldx < (1L << 23) && ldw < (1L << 23), "gemm_int8: row strides too long for 32-bit offsets");
  CWM_REQUIRE(tile >= 1 && tile <= 4, "gemm_int8: no tile %d", tile);
  const bool vector = ldy % 4 == 0 && (uintptr_t)y % 16 == 0;
#define INT8_WIDE(WM, WN)                                                                                                                           \
  {                                                                                                                                                 \
    const long m_tiles = (M + 32 * WM - 1) / (32 * WM), n_tiles = (N + 64 * WN - 1) / (64 * WN);                                                    \
    CWM_REQUIRE(m_tiles * n_tiles * (K / 128) < (1L << 31), "gemm_int8: too many steps of tiles");                                                  \
    const dim3 grid((unsigned)(m_tiles * n_tiles < units ? m_tiles * n_tiles : units));                                                             \
    if (dtype == CWM_BF16)                                                                                                                          \
      hipLaunchKernelGGL((gemm_int8_wide_kernel<WM, WN, bf16_t>), grid, dim3(512), 0, stream, (const int8_t*)X, ldx, a, (const int8_t*)W, ldw,      \
                         w_scale, bias, (bf16_t*)y, ldy, vector, M, N, K / 128, (int)m_tiles, (int)n_tiles);                                         \
    else                                                                                                                                            \
      hipLaunchKernelGGL((gemm_int8_wide_kernel<WM, WN, float>), grid, dim3(512), 0, stream, (const int8_t*)X, ldx, a, (const int8_t*)W, ldw,       \
                         w_scale, bias, (float*)y, ldy, vector, M, N, K / 128, (int)m_tiles, (int)n_tiles);                                          \
  }
  if (tile == 1) INT8_WIDE(8, 2)
  if (tile == 2) INT8_WIDE(4, 4)
  if (tile == 3) INT8_WIDE(2, 2)
  if (tile == 4) INT8_WIDE(4, 2)
  return cwm_launch_status("gemm_int8 (many rows)");
}
