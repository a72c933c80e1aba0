// Writes keys and values into the cache of 4 or 8 bits (layout and formulas: quant_cache.h) and reads them back.
//
// Both kernels take eight tokens of the list at a time, the tokens of one value block where the list follows a sequence.
// Writing, four lanes share a group, lane j with its elements 8 j .. + 7: a lane's codes of a key are one piece of memory, the
// largest and smallest of a group are two exchanges between lanes, and the two elements that a rotation turns are the lane's own.
#include "half_parts.h"
#include "quant_cache.h"

CWM_DEFINE_ERROR_API

#define HEADS_A_BLOCK 8
#define CHUNK 8  // tokens of a block

template <typename T> __device__ __forceinline__ void load8(const T* p, bool aligned, float (&x)[8]);
template <> __device__ __forceinline__ void load8<bf16_t>(const bf16_t* p, bool aligned, float (&x)[8]) {
  if (aligned) {
    const uint4 u = *(const uint4*)p;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf16_to_f32(p[e]);
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, bool aligned, float (&x)[8]) {
  if (aligned) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[e];
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, bool aligned, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<bf16_t>(bf16_t* p, bool aligned, const float (&x)[8]) {
  if (aligned) {
    *(uint4*)p = make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = f32_to_bf16(x[e]);
  }
}
template <> __device__ __forceinline__ void store8<float>(float* p, bool aligned, const float (&x)[8]) {
  if (aligned) {
    *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = x[e];
  }
}
// A number of 64 bits rounded to float32.  The empty instruction keeps the compiler from joining this rounding with one to
// bfloat16 that follows: rounded once or twice, ties fall differently.
__device__ __forceinline__ float to_float(double x) {
  float f = (float)x;
  asm volatile("" : "+v"(f));
  return f;
}
template <typename T> __device__ __forceinline__ float as_stored(float x);
template <> __device__ __forceinline__ float as_stored<bf16_t>(float x) { return bf16_to_f32(f32_to_bf16(x)); }
template <> __device__ __forceinline__ float as_stored<float>(float x) { return x; }

// N words at an address that is a multiple of 4 N bytes, in the widest pieces that allows.
template <int N> __device__ __forceinline__ void put_words(uint32_t* p, const uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *(uint4*)(p + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) *(uint2*)(p + i) = make_uint2(w[i], w[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = w[i];
  }
}
template <int N> __device__ __forceinline__ void get_words(const uint32_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 u = *(const uint4*)(p + i);
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 u = *(const uint2*)(p + i);
      w[i] = u.x, w[i + 1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p[i];
  }
}

// N numbers of one row to an address that is a multiple of their size: past the caches (the caller's next reads come from other
// compute units, and long lists are larger than the caches: 131,072 tokens of 8 heads of 128 take 169 us, 179 through them).
template <int N> __device__ __forceinline__ void stream_out(bf16_t* p, const float (&x)[N]) {
  typedef uint32_t words_t __attribute__((ext_vector_type(N / 2)));
  words_t w;
#pragma unroll
  for (int e = 0; e < N / 2; ++e) w[e] = pack2_bf16(x[2 * e], x[2 * e + 1]);
  __builtin_nontemporal_store(w, (words_t*)p);
}
template <int N> __device__ __forceinline__ void stream_out(float* p, const float (&x)[N]) {
  constexpr int M = N < 4 ? N : 4;
  typedef float floats_t __attribute__((ext_vector_type(M)));
#pragma unroll
  for (int i = 0; i < N; i += M) {
    floats_t f;
#pragma unroll
    for (int e = 0; e < M; ++e) f[e] = x[i + e];
    __builtin_nontemporal_store(f, (floats_t*)(p + i));
  }
}

// Largest and smallest of eight values; a value that is not finite makes the largest infinite.
__device__ __forceinline__ void extremes(const float (&x)[8], float& hi, float& lo) {
  float rest = 0.f;  // NaN where a value is not finite
  hi = lo = x[0];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest = fmaf(x[e], 0.f, rest), hi = fmaxf(hi, x[e]), lo = fminf(lo, x[e]);
  if (rest != 0.f) hi = __builtin_inff();
}
template <int QUAD_PERM> __device__ __forceinline__ float of_quad(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), QUAD_PERM, 15, 15, true));
}
__device__ __forceinline__ void over_lanes(float& hi, float& lo) {  // of the four lanes of a group
  hi = fmaxf(hi, of_quad<0xb1>(hi)), lo = fminf(lo, of_quad<0xb1>(lo));
  hi = fmaxf(hi, of_quad<0x4e>(hi)), lo = fminf(lo, of_quad<0x4e>(lo));
}

// a / d in 64 bits for d of 7, 15, 127 and 255: the product with the reciprocal and its remainder give the rounded quotient
// (Markstein's theorem: the reciprocals lie within 0.3 steps).
template <int d> __device__ __forceinline__ double over(double a) {
  constexpr double inv = 1. / d;
  const double q = a * inv;
  return fma(fma(-q, (double)d, a), inv, q);
}

// Step and offset of a group, in 64 bits: a step that just fits (a quotient without a remainder) is common among bfloat16
// numbers and must not be taken for the next larger one.
template <int BITS> __device__ __forceinline__ uint32_t group_word(float hi, float lo) {
  constexpr int H = 1 << (BITS - 1);
  if (hi == __builtin_inff()) return 0x7fc07fc0u;
  uint32_t z = f32_to_bf16(to_float(over<2 * H - 1>((double)H * hi + (double)(H - 1) * lo)));
  if ((z & 0x7fffu) == 0x7f80u) z -= 1;  // float32 values next to the largest one: the largest of bfloat16
  const double zd = word_offset(z);
  const float need = (float)fmax(over<H - 1>(hi - zd), (zd - lo) * (1. / H));
  return ((__float_as_uint(need) + 0xffffu) & 0xffff0000u) | z;
}

// The codes of eight numbers, less H.  float32 arithmetic decides one except next to a tie, where it may be off by its own
// rounding (the quotient is at most 2^7; a reciprocal off by 2^-23 and two roundings of 2^-24 make it, 3.1e-5 in all): there it is the quotient of 64 bits.
template <int BITS> __device__ __forceinline__ void codes_of(const float (&x)[8], uint32_t word, int (&c)[8]) {
  constexpr int H = 1 << (BITS - 1);
  const float s = word_step(word), z = word_offset(word);
  const float inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;  // a step of 0 or NaN: codes of H
  float r[8], off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (x[e] - z) * inv;
    r[e] = rintf(t);
    off = fmaxf(off, fabsf(t - r[e]));
  }
  if (off >= 0.4999f || inv == __builtin_inff()) {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = s > 0.f ? (float)rint(((double)x[e] - (double)z) / (double)s) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = min(max((int)r[e], -H), H - 1);  // a NaN gives 0
}

// A token's place in the cache: the first byte of its page and its slot, or no page.
struct Place {
  uint8_t* page;
  int slot;
};
__device__ __forceinline__ Place place_of(uint8_t* cache, long page_bytes, int pos, int seq, const int* __restrict__ block_table, int n_seqs,
                                          int table_width, int page_size, int num_pages) {
  Place p = {nullptr, 0};
  if (pos < 0 || seq < 0 || seq >= n_seqs) return p;
  const int lp = pos / page_size;
  const int page = lp < table_width ? block_table[(size_t)seq * table_width + lp] : -1;
  if (page < 0 || page >= num_pages) return p;
  p.page = cache + (size_t)page * page_bytes;
  p.slot = pos - lp * page_size;
  return p;
}

// Heads of a writing block: up to 512 lanes (4,096 tokens of 8 heads of 128 take 16.6 us, with 256 lanes 17.9, with 1,024 19.0).
__host__ __device__ constexpr int write_heads(int groups) { return 16 / groups < HEADS_A_BLOCK ? 16 / groups : HEADS_A_BLOCK; }

// grid: (chunks of eight tokens, groups of `heads_a_block` heads: those of the keys, of the values, then of the queries)
// block: a lane for eight elements: 8 tokens x heads x G groups x 4
// Prompts are bound by their arithmetic (300 instructions a lane, the turns and the rounding in 64 bits the most of them: 4,096
// tokens of 8 heads of 128 in 16.6 us, whose bytes take 5), decoded tokens by what waits for what, which the fetching of the code itself
// belongs to: with a lane for all groups of a head, four times the code, eight tokens took 7.1 us, now 5.0.  That form was the faster
// one for prompts (4,096 tokens 13.6 us); decoded tokens, which every step has, decided.  The queries' blocks make the turns
// again, one group of heads each: with 48 heads of queries 4,096 tokens take 41.6 us.
template <typename T, int G, int BITS>
__global__ void __launch_bounds__(512)
quant_kv_write_kernel(const T* __restrict__ k, long k_stride, const T* __restrict__ v, long v_stride, T* __restrict__ q, long q_stride,
                      const int* __restrict__ positions, const int* __restrict__ seq_of_token, const float* __restrict__ inv_freq,
                      uint8_t* __restrict__ cache, const int* __restrict__ block_table, int n_seqs, int table_width, int page_size, int num_pages,
                      int n_tokens, int n_kv_heads, int n_q_heads, int heads_a_block, int kv_groups, bool k_aligned, bool v_aligned, bool q_aligned) {
  constexpr int D = 32 * G;
  constexpr int MOST_HEADS = write_heads(G);
  constexpr int UNITS = BITS == 4 ? D / 2 : D;  // rows of eight bytes of a value block
  constexpr int WORDS = BITS / 4;               // of a group's eight codes
  __shared__ double turn_s[CHUNK][D / 2], turn_c[CHUNK][D / 2];
  __shared__ __attribute__((aligned(8))) uint8_t block_codes[MOST_HEADS][UNITS][8];
  __shared__ float2 block_extremes[CHUNK][MOST_HEADS][G];
  __shared__ uint8_t* dst_page[CHUNK];
  __shared__ int dst_slot[CHUNK];

  const int t0 = blockIdx.x * CHUNK;
  const int kind = blockIdx.y < kv_groups ? 0 : (blockIdx.y < 2 * kv_groups ? 1 : 2);  // keys, values, queries
  const int head0 = (blockIdx.y - kind * kv_groups) * heads_a_block;
  const int tid = threadIdx.x;
  const int j = tid & 3, g = (tid >> 2) % G, pair = tid / (4 * G), tk = pair / heads_a_block, head_in_block = pair - tk * heads_a_block;
  const int t = t0 + tk;
  const int head = head0 + head_in_block;
  const int heads = kind == 2 ? n_q_heads : n_kv_heads;
  const bool mine = t < n_tokens && head < heads;
  const QuantHead at = quant_head(page_size, D, BITS);

  // The loads of the row and of the tokens' places are under way while the turns are computed.  A lane without a row takes the last one.
  const size_t at_row = (size_t)min(t, n_tokens - 1), column = (size_t)min(head, heads - 1) * D + 32 * g + 8 * j;
  float x[8];
  load8((kind == 0 ? k + at_row * k_stride : kind == 1 ? v + at_row * v_stride : q + at_row * q_stride) + column,
        kind == 0 ? k_aligned : kind == 1 ? v_aligned : q_aligned, x);
  if (kind != 2 && tid < CHUNK) {
    Place p = {nullptr, 0};
    if (t0 + tid < n_tokens)
      p = place_of(cache, at.bytes * n_kv_heads, positions[t0 + tid], seq_of_token[t0 + tid], block_table, n_seqs, table_width, page_size, num_pages);
    dst_page[tid] = p.page;
    dst_slot[tid] = p.slot;
  }

  if (kind == 1) {
    float hi, lo;
    extremes(x, hi, lo);
    over_lanes(hi, lo);
    if (j == 0) block_extremes[tk][head_in_block][g] = make_float2(hi, lo);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float2 of = block_extremes[tk][head_in_block][i];
      hi = fmaxf(hi, of.x);
      lo = fminf(lo, of.y);
    }
    const uint32_t word = group_word<BITS>(hi, lo);
    int c[8];
    codes_of<BITS>(x, word, c);
#pragma unroll
    for (int e = 0; e < 8; e += BITS == 4 ? 2 : 1) {
      const int d = 32 * g + 8 * j + e;
      if constexpr (BITS == 4)
        block_codes[head_in_block][d / 2][tk] = (uint8_t)(c[e] + 16 * c[e + 1] + 0x88);
      else
        block_codes[head_in_block][d][tk] = (uint8_t)(c[e] + 0x80);
    }
    if (mine && j == 0 && g == 0 && dst_page[tk]) *(uint32_t*)(dst_page[tk] + (size_t)head * at.bytes + at.value_words + (size_t)dst_slot[tk] * 4) = word;
    __syncthreads();
    // Eight tokens that fill a value block are stored eight bytes at a time; tokens that do not follow one another, or that
    // begin inside a block, byte by byte.
    bool whole = dst_page[0] != nullptr && (dst_slot[0] & 7) == 0;
    for (int i = 1; i < CHUNK; ++i) whole = whole && dst_page[i] == dst_page[0] && dst_slot[i] == dst_slot[0] + i;
    const int units = min(heads_a_block, n_kv_heads - head0) * UNITS;
    if (whole) {
      uint8_t* block = dst_page[0] + (size_t)head0 * at.bytes + at.values + (size_t)(dst_slot[0] >> 3) * UNITS * 8;
      for (int i = tid; i < units; i += blockDim.x) {
        const int hb = i / UNITS, u = i - hb * UNITS;
        uint2 w = *(const uint2*)block_codes[hb][u];
        if constexpr (BITS == 4) w.x = __builtin_amdgcn_perm(w.x, w.x, 0x03010200u), w.y = __builtin_amdgcn_perm(w.y, w.y, 0x03010200u);
        *(uint2*)(block + (size_t)hb * at.bytes + u * 8) = w;
      }
    } else {
      for (int i = tid; i < units; i += blockDim.x) {
        const int hb = i / UNITS, u = i - hb * UNITS;
        const uint2 w = *(const uint2*)block_codes[hb][u];
#pragma unroll
        for (int e = 0; e < CHUNK; ++e) {
          uint8_t* page = dst_page[e];
          if (!page) continue;
          const int slot = dst_slot[e], byte = BITS == 4 ? quant_place(slot & 7) : slot & 7;
          page[(size_t)(head0 + hb) * at.bytes + at.values + ((size_t)(slot >> 3) * UNITS + u) * 8 + byte] = (uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
        }
      }
    }
    return;
  }

  if (inv_freq) {
    // the turns of the eight tokens, once for all heads of the block; in 64 bits, so that a turned key is what the formula
    // gives, rounded once
    for (int i = tid; i < CHUNK * (D / 2); i += blockDim.x) {
      const int tt = i / (D / 2), f = i - tt * (D / 2);
      if (t0 + tt < n_tokens) {
        const double turns = (double)positions[t0 + tt] * (double)inv_freq[f] * 0.15915494309189535;
        sincospi(2.0 * (turns - rint(turns)), &turn_s[tt][f], &turn_c[tt][f]);
      }
    }
  }
  __syncthreads();
  if (inv_freq) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int f = 16 * g + 4 * j + e / 2;
      const double re = x[e], im = x[e + 1], c = turn_c[tk][f], s = turn_s[tk][f];
      x[e] = as_stored<T>(to_float(re * c - im * s));
      x[e + 1] = as_stored<T>(to_float(im * c + re * s));
    }
  }
  if (kind == 2) {
    if (mine) store8(q + at_row * q_stride + column, q_aligned, x);
    return;
  }
  float hi, lo;
  extremes(x, hi, lo);
  over_lanes(hi, lo);
  const uint32_t word = group_word<BITS>(hi, lo);
  int c[8];
  codes_of<BITS>(x, word, c);
  uint8_t* const page = dst_page[tk];
  if (!mine || !page) return;
  // sums of signed codes modulo 2^32, and H on every one of them at the end: nothing is carried over
  uint32_t u[8], codes[WORDS];
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = (uint32_t)c[e];
  if constexpr (BITS == 4) {
    codes[0] = ((((((u[7] * 16 + u[5]) * 16 + u[3]) * 16 + u[1]) * 16 + u[6]) * 16 + u[4]) * 16 + u[2]) * 16 + u[0] + 0x88888888u;
  } else {
    codes[0] = ((u[3] * 256 + u[2]) * 256 + u[1]) * 256 + u[0] + 0x80808080u;
    codes[WORDS - 1] = ((u[7] * 256 + u[6]) * 256 + u[5]) * 256 + u[4] + 0x80808080u;
  }
  uint8_t* const to = page + (size_t)head * at.bytes;
  const int slot = dst_slot[tk];
  put_words<WORDS>((uint32_t*)to + (((size_t)slot * 4 + j) * G + g) * WORDS, codes);
  if (j == 0) *(uint32_t*)(to + at.key_words + ((size_t)slot * G + g) * 4) = word;
}

// Reads the tokens of a list: grid (chunks of eight tokens, groups of eight heads: keys, then values).  Bound by memory, most of it the
// written rows: neighbouring lanes write neighbouring pieces, whole cache lines an instruction (131,072 tokens of 8 heads of 128 in 4
// bits: 690 MB in 169 us, 4.1 TB/s where a plain copy has 4.85; with a lane for a token's eight elements of all groups 246).
template <typename T, int G, int BITS>
__global__ void __launch_bounds__(256)
quant_kv_read_kernel(T* __restrict__ k, T* __restrict__ v, const int* __restrict__ positions, const int* __restrict__ seq_of_token,
                     const uint8_t* __restrict__ cache, const int* __restrict__ block_table, int n_seqs, int table_width, int page_size,
                     int num_pages, int n_tokens, int n_kv_heads, int kv_groups) {
  constexpr int D = 32 * G;
  constexpr int H = 1 << (BITS - 1);
  constexpr int WORDS = BITS / 4;
  __shared__ const uint8_t* src_page[CHUNK];
  __shared__ int src_slot[CHUNK];
  __shared__ uint32_t value_words[HEADS_A_BLOCK][CHUNK];
  const int t0 = blockIdx.x * CHUNK;
  const bool values = blockIdx.y >= kv_groups;
  const int head0 = (blockIdx.y - (values ? kv_groups : 0)) * HEADS_A_BLOCK;
  const int heads = min(HEADS_A_BLOCK, n_kv_heads - head0);
  const int tid = threadIdx.x;
  const int last = min(CHUNK, n_tokens - t0) - 1;
  const QuantHead at = quant_head(page_size, D, BITS);
  if (tid < HEADS_A_BLOCK * CHUNK) {
    const int tk = tid & 7, hb = tid >> 3;
    Place p = {nullptr, 0};
    if (tk <= last)
      p = place_of((uint8_t*)cache, at.bytes * n_kv_heads, positions[t0 + tk], seq_of_token[t0 + tk], block_table, n_seqs, table_width, page_size, num_pages);
    if (hb == 0) {
      src_page[tk] = p.page;
      src_slot[tk] = p.slot;
    }
    // a token without a page reads as zeros
    if (values && hb < heads) value_words[hb][tk] = p.page ? *(const uint32_t*)(p.page + (size_t)(head0 + hb) * at.bytes + at.value_words + (size_t)p.slot * 4) : 0u;
  }
  __syncthreads();

  if (!values) {
    constexpr int PIECES = D / 8;  // of a token's key; piece 4 g + j holds the codes [j][g]
    constexpr int AT_ONCE = 4;     // pieces of a thread whose loads are under way together
    const int n = (last + 1) * heads * PIECES;
    for (int i0 = tid; i0 < n; i0 += AT_ONCE * 256) {
      uint32_t codes[AT_ONCE][WORDS] = {}, word[AT_ONCE] = {};
#pragma unroll
      for (int m = 0; m < AT_ONCE; ++m) {
        const int i = i0 + 256 * m, piece = i % PIECES, th = i / PIECES, tk = th / heads, g = piece >> 2, j = piece & 3;
        const uint8_t* page = i < n ? src_page[tk] : nullptr;
        if (!page) continue;
        const uint8_t* from = page + (size_t)(head0 + th - tk * heads) * at.bytes;
        get_words<WORDS>((const uint32_t*)from + (((size_t)src_slot[tk] * 4 + j) * G + g) * WORDS, codes[m]);
        word[m] = *(const uint32_t*)(from + at.key_words + ((size_t)src_slot[tk] * G + g) * 4);
      }
#pragma unroll
      for (int m = 0; m < AT_ONCE; ++m) {
        const int i = i0 + 256 * m, piece = i % PIECES, th = i / PIECES, tk = th / heads;
        if (i >= n) break;
        const float s = word_step(word[m]), z = word_offset(word[m]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = BITS == 4 ? (codes[m][0] >> (4 * (e / 2 + 4 * (e % 2)))) & 15 : (codes[m][e / 4 % WORDS] >> (8 * (e & 3))) & 255;
          x[e] = fmaf(s, (float)(c - H), z);
        }
        stream_out(k + ((size_t)(t0 + tk) * n_kv_heads + head0 + th - tk * heads) * D + 8 * piece, x);
      }
    }
    return;
  }

  // Tokens that follow one another lie in at most two value blocks, of which a thread reads its sixteen bytes each.
  const int lead = src_slot[0] & 7, second = min(8 - lead, last);
  bool run = src_page[0] != nullptr && src_page[second] != nullptr;
  for (int i = 1; i <= last; ++i) {
    const int first = i < 8 - lead ? 0 : second;
    run = run && src_page[i] == src_page[first] && src_slot[i] == src_slot[first] + i - first;
  }
  run = run && (second < 8 - lead || (src_slot[second] & 7) == 0);
  constexpr int DIMS = BITS == 4 ? 4 : 2;  // of a thread: sixteen bytes of a value block
  constexpr int UNITS = D / DIMS;
  for (int i = tid; i < heads * UNITS; i += blockDim.x) {
    const int hb = i / UNITS, u = i - hb * UNITS, head = head0 + hb;
    const size_t unit = (size_t)head * at.bytes + at.values + (size_t)u * 16;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (run) {
      a = b = *(const uint4*)(src_page[0] + unit + (size_t)(src_slot[0] >> 3) * (D * BITS));
      if (lead) b = *(const uint4*)(src_page[second] + unit + (size_t)(src_slot[second] >> 3) * (D * BITS));
    }
#pragma unroll
    for (int e = 0; e < CHUNK; ++e) {
      if (e > last) break;
      const uint8_t* page = src_page[e];
      const int slot = src_slot[e], place = BITS == 4 ? quant_place(slot & 7) : slot & 7;
      uint32_t byte[2] = {};
      if (run) {
        const bool in_a = e < 8 - lead;
        byte[0] = (place < 4 ? (in_a ? a.x : b.x) : (in_a ? a.y : b.y)) >> (8 * (place & 3)) & 255u;
        byte[1] = (place < 4 ? (in_a ? a.z : b.z) : (in_a ? a.w : b.w)) >> (8 * (place & 3)) & 255u;
      } else if (page) {
        const uint8_t* p = page + unit + (size_t)(slot >> 3) * (D * BITS) + place;
        byte[0] = p[0], byte[1] = p[8];
      }
      const uint32_t word = value_words[hb][e];
      const float s = word_step(word), z = word_offset(word);
      float x[DIMS];
#pragma unroll
      for (int d = 0; d < DIMS; ++d) x[d] = fmaf(s, (float)((int)(BITS == 4 ? (byte[d / 2] >> (4 * (d & 1))) & 15u : byte[d % 2]) - H), z);
      stream_out(v + ((size_t)(t0 + e) * n_kv_heads + head) * D + DIMS * u, x);
    }
  }
}

// Unpacks keys and values of whole sequences to float16 in the layout of a cache of that type, [pages][2][heads][PAGE * D], keys
// [slot][D], values [slot / 8][D][8], for an attention of many rows: its blocks would each unpack the same keys (a prompt of 2,048
// tokens with 6 query heads to a key/value head is 96 blocks a head: the two launches take 8 and 78 us, one whose blocks
// unpacked for themselves took 197).  `exponents` [pages][heads][PAGE / 32][2] has those of the
// keys and of the values of every 32 tokens (half_parts.h), by the bounds that their words set.  List item: {sequence, first key (a
// multiple of UNPACK_KEYS), page of the unpacked cache, first key that the sequence's queries read}; grid (items, heads, keys and
// values).  What a query must not read without a NaN (a key without a page, a value held as NaN) becomes a key of NaN with a value
// of zeros: a masked score takes no part, where zero times NaN would.  So does a key that a window has passed: what lies there may be
// another sequence's by now, and must not set the exponent of its 32.
#define UNPACK_KEYS 64
// the largest magnitude that a word lets its group have; a NaN counts for nothing (fmaxf)
template <int BITS> __device__ __forceinline__ float word_bound(uint32_t word) {
  constexpr float H = 1 << (BITS - 1);
  const float s = word_step(word), z = word_offset(word);
  return fmaxf(fmaxf(fabsf(fmaf(-H, s, z)), fabsf(fmaf(H - 1, s, z))), 0.f);
}
template <int G, int BITS>
__global__ void __launch_bounds__(256)
quant_unpack_kernel(uint16_t* __restrict__ out, int* __restrict__ exponents, int out_page, const int* __restrict__ list, const uint8_t* __restrict__ cache,
                    const int* __restrict__ block_table, int table_width, int page_size, int num_pages, const int* __restrict__ kv_len, int n_kv_heads) {
  constexpr int D = 32 * G;
  constexpr int UNITS = BITS == 4 ? D / 2 : D;
  constexpr int H = 1 << (BITS - 1);
  constexpr int WORDS = BITS / 4;
  __shared__ float tops[UNPACK_KEYS / 16];
  const int* item = list + (size_t)blockIdx.x * 4;
  const int b = item[0], key0 = item[1], first = item[3], head = blockIdx.y;
  const int end = kv_len[b];
  const QuantHead at = quant_head(page_size, D, BITS);
  const size_t plane = (size_t)n_kv_heads * out_page * D;
  uint16_t* to = out + (size_t)item[2] * 2 * plane + (size_t)head * out_page * D;
  const int slot0 = key0 % out_page;
  int* exponents_to = exponents + (((size_t)item[2] * n_kv_heads + head) * (out_page / 32) + slot0 / 32) * 2;
  auto page_of = [&](int key, int& slot) -> const uint8_t* {  // the head's first byte in the key's page
    const int lp = key / page_size;
    slot = key - lp * page_size;
    const int page = lp < table_width ? block_table[(size_t)b * table_width + lp] : -1;
    return page >= 0 && page < num_pages ? cache + ((size_t)page * n_kv_heads + head) * at.bytes : nullptr;
  };
  auto put8 = [](uint16_t* p, const float(&x)[8]) {
    *(uint4*)p = make_uint4(pack2_f16(x[0], x[1]), pack2_f16(x[2], x[3]), pack2_f16(x[4], x[5]), pack2_f16(x[6], x[7]));
  };
  const int wave = threadIdx.x >> 6;
  if (blockIdx.z == 0) {
    const int key = key0 + (threadIdx.x >> 2), j = threadIdx.x & 3;
    int slot;
    const uint8_t* from = key >= first && key < end ? page_of(key, slot) : nullptr;
    uint32_t codes[G * WORDS] = {}, words[G];
    const bool held = from != nullptr;
    bool bad = !held;
    float most = 0.f;
    if (held) {
      get_words<G * WORDS>((const uint32_t*)from + ((size_t)slot * 4 + j) * G * WORDS, codes);
      get_words<G>((const uint32_t*)(from + at.key_words) + (size_t)slot * G, words);
      const float vs = word_step(*(const uint32_t*)(from + at.value_words + (size_t)slot * 4));
      bad = vs != vs;
#pragma unroll
      for (int g = 0; g < G; ++g) most = fmaxf(most, word_bound<BITS>(words[g]));
    }
    most = wave_max(most);
    if ((threadIdx.x & 63) == 0) tops[wave] = most;
    __syncthreads();
    const int e = half_exponent(fmaxf(tops[wave & ~1], tops[wave | 1]));  // 16 keys a wavefront
    if ((threadIdx.x & 127) == 0) exponents_to[(threadIdx.x >> 7) * 2] = e;
    if (key >= end) return;
    const float down = power_of_two(-e);
    uint16_t* row = to + (size_t)(slot0 + (threadIdx.x >> 2)) * D + 8 * j;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float s = bad ? __uint_as_float(0x7fc00000u) : word_step(words[g]), z = bad ? s : word_offset(words[g]);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = BITS == 4 ? (codes[g] >> (4 * (i / 2 + 4 * (i % 2)))) & 15 : (codes[(2 * g + i / 4) % (G * WORDS)] >> (8 * (i & 3))) & 255;
        x[i] = fmaf(s, (float)(c - H), z) * down;
      }
      put8(row + 32 * g, x);
    }
    return;
  }
  if (threadIdx.x < UNPACK_KEYS) {
    const int key = key0 + threadIdx.x;
    int slot;
    const uint8_t* from = key >= first && key < end ? page_of(key, slot) : nullptr;
    float most = from ? word_bound<BITS>(*(const uint32_t*)(from + at.value_words + (size_t)slot * 4)) : 0.f;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
    if ((threadIdx.x & 31) == 0) {
      tops[threadIdx.x >> 5] = most;
      exponents_to[(threadIdx.x >> 5) * 2 + 1] = half_exponent(most, VALUES_LEAST);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < UNPACK_KEYS / 8 * UNITS; i += 256) {
    const int block = i / UNITS, u = i - block * UNITS, key = key0 + 8 * block;
    if (key >= end) return;
    int slot;
    const uint8_t* from = page_of(key, slot);
    uint2 codes = make_uint2(0, 0);
    uint32_t words[8] = {};
    if (from) {
      codes = *(const uint2*)(from + at.values + ((size_t)(slot >> 3) * UNITS + u) * 8);
      get_words<8>((const uint32_t*)(from + at.value_words) + slot, words);
    }
    const float down = power_of_two(-half_exponent(tops[block >> 2], VALUES_LEAST));
    float x[BITS == 4 ? 2 : 1][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int place = BITS == 4 ? (e & 4) | ((e & 1) << 1) | ((e >> 1) & 1) : e;
      const int c = ((place < 4 ? codes.x : codes.y) >> (8 * (place & 3))) & 255;
      const float s = word_step(words[e]), z = word_offset(words[e]);
      const bool none = s != s || key + e < first;
      if constexpr (BITS == 4) {
        x[0][e] = none ? 0.f : fmaf(s, (float)((c & 15) - H), z) * down;
        x[1][e] = none ? 0.f : fmaf(s, (float)((c >> 4) - H), z) * down;
      } else {
        x[0][e] = none ? 0.f : fmaf(s, (float)(c - H), z) * down;
      }
    }
    uint16_t* row = to + plane + ((size_t)((slot0 >> 3) + block) * D + (BITS == 4 ? 2 * u : u)) * 8;
    put8(row, x[0]);
    if constexpr (BITS == 4) put8(row + 8, x[BITS == 4 ? 1 : 0]);
  }
}

// ---- entry points ------------------------------------------------------------------------ //
#define FOR_GROUPS(CALL, BITS)     \
  switch (head_dim / 32) {         \
    case 1: CALL(1, BITS); break;  \
    case 2: CALL(2, BITS); break;  \
    case 3: CALL(3, BITS); break;  \
    case 4: CALL(4, BITS); break;  \
    case 5: CALL(5, BITS); break;  \
    case 6: CALL(6, BITS); break;  \
    case 7: CALL(7, BITS); break;  \
    default: CALL(8, BITS); break; \
  }

extern "C" int cwm_quant_kv_write(const void* k, long k_stride, const void* v, long v_stride, void* q, long q_stride, int dtype, const int* positions,
                                  const int* seq_of_token, const float* inv_freq, void* cache, const int* block_table, int n_seqs, int table_width,
                                  int page_size, int num_pages, int n_tokens, int n_kv_heads, int n_q_heads, int head_dim, int bits,
                                  hipStream_t stream) {
  QUANT_REQUIRE_SIZES("quant_kv_write");
  CWM_REQUIRE(n_tokens >= 0 && n_q_heads >= 0 && n_seqs >= 0, "quant_kv_write: negative sizes");
  if (n_tokens == 0) return 0;
  CWM_REQUIRE(k && v && cache && block_table && positions && seq_of_token, "quant_kv_write: a tensor is missing");
  CWM_REQUIRE(q || n_q_heads == 0, "quant_kv_write: queries missing");
  CWM_REQUIRE(((uintptr_t)cache % 16) == 0, "quant_kv_write: the cache must be 16-byte aligned");
  const int groups = head_dim / 32, chunks = (n_tokens + CHUNK - 1) / CHUNK;
  const int heads = q && n_q_heads > n_kv_heads ? n_q_heads : n_kv_heads, heads_a_block = write_heads(groups) < heads ? write_heads(groups) : heads;
  const int kv_groups = (n_kv_heads + heads_a_block - 1) / heads_a_block;
  const int q_groups = q && inv_freq ? (n_q_heads + heads_a_block - 1) / heads_a_block : 0;
  CWM_REQUIRE(2 * kv_groups + q_groups <= 65535, "quant_kv_write: too many heads");
  const dim3 grid(chunks, 2 * kv_groups + q_groups), block(32 * groups * heads_a_block);
  const int piece = dtype == CWM_BF16 ? 8 : 4;
  const bool ka = k_stride % piece == 0 && (uintptr_t)k % 16 == 0, va = v_stride % piece == 0 && (uintptr_t)v % 16 == 0;
  const bool qa = q_stride % piece == 0 && (uintptr_t)q % 16 == 0;
#define CALL_WRITE(G, BITS)                                                                                                                      \
  if (dtype == CWM_BF16)                                                                                                                         \
    hipLaunchKernelGGL((quant_kv_write_kernel<bf16_t, G, BITS>), grid, block, 0, stream, (const bf16_t*)k, k_stride, (const bf16_t*)v, v_stride, \
      (bf16_t*)q, q_stride, positions, seq_of_token, inv_freq, (uint8_t*)cache, block_table, n_seqs, table_width, page_size,                     \
      num_pages, n_tokens, n_kv_heads, n_q_heads, heads_a_block, kv_groups, ka, va, qa);                                                                        \
  else                                                                                                                                           \
    hipLaunchKernelGGL((quant_kv_write_kernel<float, G, BITS>), grid, block, 0, stream, (const float*)k, k_stride, (const float*)v, v_stride,    \
      (float*)q, q_stride, positions, seq_of_token, inv_freq, (uint8_t*)cache, block_table, n_seqs, table_width, page_size,                      \
      num_pages, n_tokens, n_kv_heads, n_q_heads, heads_a_block, kv_groups, ka, va, qa)
  if (bits == 4) {
    FOR_GROUPS(CALL_WRITE, 4)
  } else {
    FOR_GROUPS(CALL_WRITE, 8)
  }
  return cwm_launch_status("quant_kv_write");
}

extern "C" int cwm_quant_kv_read(void* k, void* v, int dtype, const int* positions, const int* seq_of_token, const void* cache, const int* block_table,
                                 int n_seqs, int table_width, int page_size, int num_pages, int n_tokens, int n_kv_heads, int head_dim, int bits,
                                 hipStream_t stream) {
  QUANT_REQUIRE_SIZES("quant_kv_read");
  CWM_REQUIRE(n_tokens >= 0 && n_seqs >= 0, "quant_kv_read: negative sizes");
  if (n_tokens == 0) return 0;
  CWM_REQUIRE(k && v && cache && block_table && positions && seq_of_token, "quant_kv_read: a tensor is missing");
  CWM_REQUIRE(((uintptr_t)cache % 16) == 0 && ((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0, "quant_kv_read: tensors must be 16-byte aligned");
  const int kv_groups = (n_kv_heads + HEADS_A_BLOCK - 1) / HEADS_A_BLOCK;
  CWM_REQUIRE(2 * kv_groups <= 65535, "quant_kv_read: too many heads");
  const dim3 grid((n_tokens + CHUNK - 1) / CHUNK, 2 * kv_groups), block(256);
#define CALL_READ(G, BITS)                                                                                                               \
  if (dtype == CWM_BF16)                                                                                                                 \
    hipLaunchKernelGGL((quant_kv_read_kernel<bf16_t, G, BITS>), grid, block, 0, stream, (bf16_t*)k, (bf16_t*)v, positions, seq_of_token, \
      (const uint8_t*)cache, block_table, n_seqs, table_width, page_size, num_pages, n_tokens, n_kv_heads, kv_groups);                   \
  else                                                                                                                                   \
    hipLaunchKernelGGL((quant_kv_read_kernel<float, G, BITS>), grid, block, 0, stream, (float*)k, (float*)v, positions, seq_of_token,    \
      (const uint8_t*)cache, block_table, n_seqs, table_width, page_size, num_pages, n_tokens, n_kv_heads, kv_groups)
  if (bits == 4) {
    FOR_GROUPS(CALL_READ, 4)
  } else {
    FOR_GROUPS(CALL_READ, 8)
  }
  return cwm_launch_status("quant_kv_read");
}

extern "C" int cwm_quant_unpack(void* out, int* exponents, int out_page, const int* list, int n_items, const void* cache, const int* block_table, int table_width,
                                int page_size, int num_pages, const int* kv_len, int n_kv_heads, int head_dim, int bits, hipStream_t stream) {
  QUANT_REQUIRE_SIZES("quant_unpack");
  CWM_REQUIRE(n_items >= 0 && n_kv_heads <= 65535 && out_page > 0 && out_page % UNPACK_KEYS == 0, "quant_unpack: bad sizes");
  if (n_items == 0) return 0;
  CWM_REQUIRE(out && exponents && list && cache && block_table && kv_len, "quant_unpack: a tensor is missing");
  CWM_REQUIRE((uintptr_t)cache % 16 == 0 && (uintptr_t)out % 16 == 0, "quant_unpack: tensors must be 16-byte aligned");
  const dim3 grid(n_items, n_kv_heads, 2);
#define CALL_UNPACK(G, BITS)                                                                                                                   \
  hipLaunchKernelGGL((quant_unpack_kernel<G, BITS>), grid, dim3(256), 0, stream, (uint16_t*)out, exponents, out_page, list, (const uint8_t*)cache, \
                     block_table, table_width, page_size, num_pages, kv_len, n_kv_heads)
  if (bits == 4) {
    FOR_GROUPS(CALL_UNPACK, 4)
  } else {
    FOR_GROUPS(CALL_UNPACK, 8)
  }
  return cwm_launch_status("quant_unpack");
}
