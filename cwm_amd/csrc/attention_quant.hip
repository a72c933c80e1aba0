// Paged causal attention over a cache held in 4 or 8 bits (layout and formulas: quant_cache.h), on the matrix cores, for
// decoded tokens and prompt portions in one launch.  Compiled per head size: -DHEAD_DIM=<multiple of 32, at most 256>.
//
// The query at position p reads keys max(0, p - window_left) .. p; scores scale (q . k), softmax, sum of the values; query
// head h reads key/value head h / (Hq / Hkv).  Rows are (new token, query head of the group) pairs, 16 to a tile; work items
// as of the attention over a cache in the activations' type: {sequence, first row, first key, end key, partial slot or -1, 0}.
//
// Codes go to the matrix instruction as they are: a code of 4 bits under the exponent of 128 is the bfloat16 number 128 + c,
// one mask and one "or" for two of them, and exact.  With the key k_d = z_g + s_g (c_d - H) of group g of 32 elements,
//     q . k = sum_g s_g (sum_d q_d (OFF' + c_d)) + sum_g (z_g - OFF s_g) sum_d q_d,   OFF = OFF' + H
// where the second sum is one more matrix product, of the words (offset, step) of a key, which are already pairs of
// bfloat16 numbers in a register, with the query's sums in three bfloat16 parts; and a product of the words with a column
// that is 1 at one place brings a group's step to the lanes that hold its scores.  No vector instruction touches a word.
//     o = sum_j p_j v_j = sum_j b_j (OFF' + c_j) - OFF sum_j b_j + sum_j p_j z_j,   b_j = p_j s_j in two bfloat16 parts
// The sum of the b_j is one more matrix product (a row of ones), so that it holds the same rounded numbers; the last sum is
// kept in float32.  One part would round the weights to 2^-8 of themselves, as much as the result is rounded; the second takes
// that to 2^-16 for 2 us of 60 (the step below), since the matrix cores wait for the cache.
// float32 queries: q and b in three bfloat16 parts each, codes without an offset (c - H is exact in bfloat16).
//
// Decoded tokens are bound by the reading of the cache: eight sequences of 32,768 tokens, 48 query heads on 8 of 128, 4 bits: 310 MB in
// 62 us (5.0 TB/s; a plain read has 6.9) and 5 for joining the chunks; in bfloat16 the same step reads 1,074 MB in 178 (6.0 TB/s).  A wavefront's
// loads run two tiles ahead of its arithmetic; eight wavefronts a block instead of four take 77 us.  A step of few keys is bound by its
// latencies (1,000 keys: 11.4 us).
//
// Lanes as in the attention over a bfloat16 cache (lane 16 j + n): S^T = K Q^T leaves lane (row n, j) the keys 8 j .. 8 j + 7
// of 32, which is the operand of O^T = V^T P^T, so probabilities never move.
#include "quant_cache.h"
#include "three_parts.h"

CWM_DEFINE_ERROR_API

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
#if HEAD_DIM % 32 != 0 || HEAD_DIM > 256 || HEAD_DIM < 32
#error "HEAD_DIM must be a multiple of 32 between 32 and 256"
#endif

#define G (HEAD_DIM / 32)  // groups of a key
#define QUADS ((G + 3) / 4)  // operands that a key's words fill, four words each
#define D_TILES (HEAD_DIM / 16)
#define WORK_INTS 6
#define PARTIAL_STRIDE (HEAD_DIM + 4)  // reference maximum and sum after the output
#define TEAM 4  // wavefronts of a block

typedef const __attribute__((address_space(4))) int* scalar_ints;  // a uniform index is read by a scalar load

// N words at an address that is a multiple of 4 bytes, in the widest pieces.
template <int N> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  const void* from = __builtin_assume_aligned(p, 4);
  constexpr int FOURS = N / 4 * 4;
#pragma unroll
  for (int i = 0; i < FOURS; i += 4) __builtin_memcpy(&w[i], (const uint8_t*)from + 4 * i, 16);
  if constexpr (N > FOURS) __builtin_memcpy(&w[FOURS], (const uint8_t*)from + 4 * FOURS, 4 * (N - FOURS));
}

// The same through a buffer resource, which bounds the offsets: past its size a load gives zeros and reads nothing, so one of size
// 0 takes the place of a branch around the loads.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int N> __device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t r, uint32_t offset, uint32_t (&w)[N]) {
  constexpr int ONCE = 2;  // non-temporal: every block reads keys and values of its own
  constexpr int FOURS = N / 4 * 4;
#pragma unroll
  for (int i = 0; i < FOURS; i += 4) {
    const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(r, offset + 4 * i, 0, ONCE);
    w[i] = u[0], w[i + 1] = u[1], w[i + 2] = u[2], w[i + 3] = u[3];
  }
  if constexpr (N - FOURS == 3) {
    const u32x3 u = __builtin_amdgcn_raw_buffer_load_b96(r, offset + 4 * FOURS, 0, ONCE);
    w[FOURS] = u[0], w[FOURS + 1] = u[1], w[FOURS + 2] = u[2];
  } else if constexpr (N - FOURS == 2) {
    const u32x2 u = __builtin_amdgcn_raw_buffer_load_b64(r, offset + 4 * FOURS, 0, ONCE);
    w[FOURS] = u[0], w[FOURS + 1] = u[1];
  } else if constexpr (N - FOURS == 1) {
    w[FOURS] = __builtin_amdgcn_raw_buffer_load_b32(r, offset + 4 * FOURS, 0, ONCE);
  }
}

// How codes become numbers of bfloat16.  EXACT: c - H.  Else OFF' + c, OFF' = 128 for 4 bits and 0 for 8.
template <int BITS, bool EXACT> struct Codes {
  static constexpr int H = 1 << (BITS - 1);
  static constexpr float OFF = EXACT ? 0.f : (BITS == 4 ? 128.f + H : (float)H);
  // The constants of `nibbles` in registers that the compiler knows nothing of: it then forms one instruction of mask and "or", which
  // takes no two literals.  (Not one written by hand: it could not see to the wait between that and the matrix instruction.)
  uint32_t mask = 0x000f000fu, base = 0x43004300u;
  __device__ __forceinline__ Codes() { asm volatile("" : "+s"(mask), "+v"(base)); }
  // four bits from bit 0 and from bit 16 on
  __device__ __forceinline__ uint32_t nibbles(uint32_t w) const {
    if constexpr (EXACT) {
      const float a = (float)((int)(w & 15u) - H), b = (float)((int)((w >> 16) & 15u) - H);
      return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    return (w & mask) | base;
  }
  __device__ __forceinline__ uint32_t bytes(uint32_t w, int first) const {  // bytes `first` and `first + 1`
    float a = (float)((w >> (8 * first)) & 255u), b = (float)((w >> (8 * first + 8)) & 255u);
    if constexpr (EXACT) a -= H, b -= H;
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
};

// What a wavefront loads of 32 keys: lane (n, j) the codes [j] of keys 8 (n / 4) + n % 4 and + 4 with their words, and of the
// values of keys 8 j .. 8 j + 7 those of its dimensions, with their words.
template <int BITS> struct KeyTile {
  static constexpr int KC = G * BITS / 4;
  // words of the values' codes: pieces of 16 bytes (four dimensions of 4 bits, two of 8), a last one of 8 where 32 dimensions are left
  static constexpr int VC = BITS == 4 ? 2 * G : 4 * G;
  uint32_t kc[2][KC], kw[2][4 * QUADS], vc[VC], vw[8];  // zeros behind the words of a key
};

__device__ __forceinline__ float not_a_number() { return __uint_as_float(0x7fc00000u); }

// Whether any key of [first_key, last_key] lies in a logical page whose table entry is no page of the pool.
__device__ __forceinline__ bool span_lacks_page(const int* __restrict__ table, int table_width, int num_pages, int page_size, int first_key,
                                                int last_key, int lane) {
  bool bad = false;
  if (last_key >= first_key && first_key >= 0) {
    for (int lp = first_key / page_size + lane; lp <= last_key / page_size; lp += 64) {
      const int page = lp < table_width ? table[lp] : -1;
      bad = bad || (unsigned)page >= (unsigned)num_pages;
    }
  }
  return __any(bad);
}

// RT row tiles a wavefront.  SPLIT: the block's wavefronts share 16 RT rows and take the item's tiles of 32 keys in turn, and
// join their results through LDS; else each has rows of its own and walks all of the item's keys.
template <typename T, int BITS, int RT, bool SPLIT, bool PAGE32>
__global__ void __launch_bounds__(256, SPLIT ? 2 : 1)
attention_quant_kernel(const T* __restrict__ q, long q_stride, T* __restrict__ out, long out_stride, const uint8_t* __restrict__ cache,
                       const int* __restrict__ block_table, int table_width, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
                       const int* __restrict__ work, float* __restrict__ partial, int n_q_heads, int n_kv_heads, int page_size, int page_shift,
                       int num_pages, int window_left, float scale_log2e) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int PARTS = EXACT ? 3 : 1;
  constexpr int B_PARTS = EXACT ? 3 : 2;  // of a weight
  typedef Codes<BITS, EXACT> C;
  typedef KeyTile<BITS> Keys;
  const float neg_inf = -__builtin_inff();

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / n_kv_heads;
  const int g0 = blockIdx.x - item * n_kv_heads;  // key/value head
  const int* w = work + (size_t)item * WORK_INTS;
  const int b = w[0], key_begin = w[2], key_end = w[3], slot = w[4], n_chunks = w[5];
  if (key_begin >= key_end) return;  // a null item: a list of a fixed length is filled up with them

  const int group = n_q_heads / n_kv_heads;
  const int q0 = cu_q[b];
  const int n_new = cu_q[b + 1] - q0;
  const int n_old = kv_len[b] - n_new;
  const int n_rows = n_new * group;
  const int n = lane & 15, j = lane >> 4;

  bool row_valid[RT];
  int ti[RT], hq[RT], row_end[RT], row_start[RT];
  Frag8 qf[RT][PARTS][G], qs[RT][QUADS];
  Frag8 ones;  // a row of ones
  ones.u = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  const float4v zero = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = w[1] + 16 * (SPLIT ? rt : RT * wave + rt) + n;
    row_valid[rt] = r < n_rows;
    ti[rt] = row_valid[rt] ? r / group : 0;
    hq[rt] = g0 * group + (row_valid[rt] ? r - ti[rt] * group : 0);
    row_end[rt] = n_old + ti[rt];
    row_start[rt] = window_left >= 0 ? max(0, row_end[rt] - window_left) : 0;

    // queries: the B operands, and the sums over a group's elements in three parts, one part for each j < 3
    const T* qrow = q + (size_t)(q0 + ti[rt]) * q_stride + (size_t)hq[rt] * HEAD_DIM + 8 * j;
    float sum[G];  // a product with the row of ones
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if constexpr (EXACT) {
        float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
        if (row_valid[rt]) lo = *(const float4*)(qrow + 32 * g), hi = *(const float4*)(qrow + 32 * g + 4);
        const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        Frag8 part[3];
        three_parts(x, part);
        qf[rt][0][g] = part[0], qf[rt][1 % PARTS][g] = part[1], qf[rt][2 % PARTS][g] = part[2];
      } else {
        qf[rt][0][g].u = row_valid[rt] ? *(const uint4*)(qrow + 32 * g) : make_uint4(0, 0, 0, 0);
      }
      float4v d = zero;
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, qf[rt][p][g].v, d, 0, 0, 0);
      sum[g] = d[0];
    }
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = 4 * u + i < G ? sum[(4 * u + i) % G] : 0.f;
        x[2 * i + 1] = -C::OFF * x[2 * i];
      }
      Frag8 part[3];
      three_parts(x, part);
      qs[rt][u].u = j == 0 ? part[0].u : j == 1 ? part[1].u : j == 2 ? part[2].u : make_uint4(0, 0, 0, 0);
    }
  }
  // The span of keys that any of the wavefront's rows reads, and the span that all of them read: tiles within it need no masks.  Rows
  // that do not exist have queries of zeros and are not stored: they read whatever the others do.
  int lo_any = 0x7fffffff, hi_any = -1, lo_all = 0, hi_all = 0x7fffffff;
  const int first_row = w[1] + (SPLIT ? 0 : 16 * RT * wave), last_row = min(first_row + 16 * RT, n_rows) - 1;
  if (first_row <= last_row) {
    const int first_end = n_old + first_row / group, last_end = n_old + last_row / group;
    lo_any = max(key_begin, window_left >= 0 ? first_end - window_left : 0);
    hi_any = min(key_end - 1, last_end);
    lo_all = max(key_begin, window_left >= 0 ? last_end - window_left : 0);
    hi_all = min(key_end - 1, first_end);
  }
  // a row reads its keys first .. first + count - 1 of the item
  int first_key[RT];
  unsigned key_count[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    first_key[rt] = max(row_start[rt], key_begin);
    key_count[rt] = row_valid[rt] ? max(0, min(row_end[rt], key_end - 1) - first_key[rt] + 1) : 0;
  }

  const int* table = block_table + (size_t)b * table_width;
  const scalar_ints table_s = (scalar_ints)table;
  const bool page_missing = span_lacks_page(table, table_width, num_pages, page_size, lo_any, hi_any, lane);
  const QuantHead at = quant_head(page_size, HEAD_DIM, BITS);
  // a head of a page has less than 2 GiB: offsets within it are 32 bits, beside a page's address in scalar registers
  const uint32_t values_at = (uint32_t)at.values, key_words_at = (uint32_t)at.key_words, value_words_at = (uint32_t)at.value_words;
  const size_t page_bytes = (size_t)at.bytes * n_kv_heads;
  const uint8_t* base = cache + (size_t)at.bytes * g0;

  // The operands that bring a group's step out of a pair of words to all columns (1 at the upper half of the first or of the second
  // word, in one lane of four).
  typedef short Pair __attribute__((ext_vector_type(4)));
  const uint32_t one = j == 0 ? 0x3f800000u : 0u;
  const Pair pick[2] = {__builtin_bit_cast(Pair, make_uint2(one, 0)), __builtin_bit_cast(Pair, make_uint2(0, one))};
  const C codes;

  // the table's entry for a key; keys outside the item and slots without a page read page 0 and are masked
  auto entry_of = [&](int key) -> int {
    const int lp = page_shift >= 0 ? (key >> page_shift) : (key / page_size);
    return key < key_end && lp < table_width ? table[lp] : 0;
  };
  const int krel = 8 * (n >> 2) + (n & 3);
  // As many tiles' registers as there is room for: three in the lightest case, else two where they fit beside sums and queries (by
  // count, with 60 for the rest), else one, whose loads the other wavefronts' work hides (16,384 tokens of 8 heads of 256 in 8 bits,
  // batch 8: 123 us, with two that spill 306; heads of 160, where two fit: 87 and, with one, 91).
  constexpr int TILE_WORDS = 2 * Keys::KC + 2 * G + Keys::VC + 8, OTHER_WORDS = RT * (4 * D_TILES + 4 * G * PARTS) + 60;
  constexpr int BUFFERS = PAGE32 && BITS == 4 && !EXACT && HEAD_DIM <= 128 ? 3 : 2 * TILE_WORDS + OTHER_WORDS <= (SPLIT ? 240 : 320) ? 2 : 1;
  constexpr int STEP = SPLIT ? TEAM : 1;  // wavefront w starts at the item's tile w and goes on in steps of TEAM tiles, or takes every tile
  // PAGE32: a tile lies in one page, whose number is read as a scalar a tile ahead; else a lane's two are, of its keys and of its values
  auto look_up = [&](int kt) -> int {
    const int lp = min(page_shift >= 0 ? (kt >> page_shift) : (kt / page_size), table_width - 1);
    return PAGE32 ? table_s[lp] : 0;
  };
  int page_ahead = 0, k_ahead = 0, v_ahead = 0;
  const int tile0 = key_begin >> 5, tiles = ((key_end + 31) >> 5) - tile0;
  // the loads of the item's tile `t`, which may lie past its last one: then of nothing
  auto issue = [&](Keys& L, int t) {
    const int kt = 32 * (tile0 + t);
    constexpr int PIECES = Keys::VC / 4;
    if constexpr (PAGE32) {
      const int lp = page_shift >= 0 ? (kt >> page_shift) : (kt / page_size);
      const int page = (unsigned)page_ahead < (unsigned)num_pages ? page_ahead : 0;
      page_ahead = look_up(kt + 32 * STEP);
      const __amdgpu_buffer_rsrc_t head =
          __builtin_amdgcn_make_buffer_rsrc((void*)(base + (size_t)page * page_bytes), 0, t < tiles ? (int)at.bytes : 0, 0x00027000);
      const int ks = kt - lp * page_size + krel, vs = kt - lp * page_size + 8 * j;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_words<Keys::KC>(head, (uint32_t)(((ks + 4 * i) * 4 + j) * (Keys::KC * 4)), L.kc[i]);
        uint32_t words[G];
        load_words<G>(head, key_words_at + (uint32_t)(ks + 4 * i) * (G * 4), words);
#pragma unroll
        for (int g = 0; g < 4 * QUADS; ++g) L.kw[i][g] = g < G ? words[g % G] : 0u;
      }
      load_words<8>(head, value_words_at + (uint32_t)vs * 4, L.vw);
      const uint32_t vb = values_at + (uint32_t)(vs >> 3) * (HEAD_DIM * BITS);
#pragma unroll
      for (int c = 0; c < PIECES; ++c) load_words<4>(head, vb + 256 * c + 16 * n, *(uint32_t(*)[4])&L.vc[4 * c]);
      if constexpr (Keys::VC % 4 != 0) load_words<2>(head, vb + 256 * PIECES + 8 * n, *(uint32_t(*)[2])&L.vc[4 * PIECES]);
    } else {
      const int kk = kt + krel, vk = kt + 8 * j;
      const int ks = page_shift >= 0 ? kk & (page_size - 1) : kk % page_size, vs = page_shift >= 0 ? vk & (page_size - 1) : vk % page_size;
      const uint8_t* kpage = base + (size_t)((unsigned)k_ahead < (unsigned)num_pages ? k_ahead : 0) * page_bytes;
      const uint8_t* vpage = base + (size_t)((unsigned)v_ahead < (unsigned)num_pages ? v_ahead : 0) * page_bytes;
      k_ahead = entry_of(kk + 32 * STEP), v_ahead = entry_of(vk + 32 * STEP);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_words<Keys::KC>(kpage + (uint32_t)(((ks + 4 * i) * 4 + j) * (Keys::KC * 4)), L.kc[i]);
        uint32_t words[G];
        load_words<G>(kpage + (key_words_at + (uint32_t)(ks + 4 * i) * (G * 4)), words);
#pragma unroll
        for (int g = 0; g < 4 * QUADS; ++g) L.kw[i][g] = g < G ? words[g % G] : 0u;
      }
      load_words<8>(vpage + (value_words_at + (uint32_t)vs * 4), L.vw);
      const uint32_t vb = values_at + (uint32_t)(vs >> 3) * (HEAD_DIM * BITS);
#pragma unroll
      for (int c = 0; c < PIECES; ++c) load_words<4>(vpage + (vb + 256 * c + 16 * n), *(uint32_t(*)[4])&L.vc[4 * c]);
      if constexpr (Keys::VC % 4 != 0) load_words<2>(vpage + (vb + 256 * PIECES + 8 * n), *(uint32_t(*)[2])&L.vc[4 * PIECES]);
    }
  };

  float4v acc[RT][D_TILES], bsum[RT];
  float m_run[RT], neg_mc[RT], l_run[RT], z_run[RT];
  const float lazy_raw = 8.0f / scale_log2e;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int d = 0; d < D_TILES; ++d) acc[rt][d] = (float4v){0.f, 0.f, 0.f, 0.f};
    bsum[rt] = (float4v){0.f, 0.f, 0.f, 0.f};
    m_run[rt] = neg_inf, neg_mc[rt] = 0.f, l_run[rt] = 0.f, z_run[rt] = 0.f;
  }

  auto compute = [&](const Keys& L, int kt) {
    float4v st[RT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      Frag8 words[QUADS];
#pragma unroll
      for (int u = 0; u < QUADS; ++u)
        words[u].u = make_uint4(L.kw[t][4 * u], L.kw[t][4 * u + 1], L.kw[t][4 * u + 2], L.kw[t][4 * u + 3]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        st[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(words[0].v, qs[rt][0].v, zero, 0, 0, 0);
        if constexpr (QUADS > 1) st[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(words[QUADS - 1].v, qs[rt][QUADS - 1].v, st[rt][t], 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        Frag8 kf;
        if constexpr (BITS == 4) {
          const uint32_t c = L.kc[t][g % Keys::KC];
          kf.u = make_uint4(codes.nibbles(c), codes.nibbles(c >> 4), codes.nibbles(c >> 8), codes.nibbles(c >> 12));
        } else {
          const uint32_t c0 = L.kc[t][(2 * g) % Keys::KC], c1 = L.kc[t][(2 * g + 1) % Keys::KC];
          kf.u = make_uint4(codes.bytes(c0, 0), codes.bytes(c0, 2), codes.bytes(c1, 0), codes.bytes(c1, 2));
        }
        const uint2 pair = make_uint2(L.kw[t][g / 2 * 2], L.kw[t][g / 2 * 2 + 1]);
        const float4v step = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(Pair, pair), pick[g % 2], zero, 0, 0, 0);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float4v d = zero;
#pragma unroll
          for (int p = PARTS - 1; p >= 0; --p) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf.v, qf[rt][p][g].v, d, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) st[rt][t][i] = fmaf(step[i], d[i], st[rt][t][i]);
        }
      }
    }
    const bool need_mask = kt < lo_all || kt + 31 > hi_all;
    Frag8 bf[RT][B_PARTS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8] = {st[rt][0][0], st[rt][0][1], st[rt][0][2], st[rt][0][3], st[rt][1][0], st[rt][1][1], st[rt][1][2], st[rt][1][3]};
      uint32_t hidden = 0;
      if (need_mask) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool ok = (unsigned)(kt + 8 * j + e - first_key[rt]) < key_count[rt];
          hidden |= ok ? 0u : 1u << e;
          x[e] = ok ? x[e] : neg_inf;
        }
      }
#define MAXIMUM(a, b) __builtin_elementwise_maximum(a, b)
      float top = MAXIMUM(MAXIMUM(MAXIMUM(x[0], x[1]), MAXIMUM(x[2], x[3])), MAXIMUM(MAXIMUM(x[4], x[5]), MAXIMUM(x[6], x[7])));
      // m is a reference, not the maximum: it moves, and what has been summed is rescaled, when a row's scores outgrow it by
      // a factor of 256 in p
      if (__any(top - m_run[rt] > lazy_raw)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float highest = fmaxf(m_run[rt], top);
        const float m_new = highest - m_run[rt] > lazy_raw ? highest : m_run[rt];
        const float neg = m_new == neg_inf ? 0.f : -m_new * scale_log2e;
        const float alpha = __builtin_amdgcn_exp2f(fmaf(m_run[rt], scale_log2e, neg));
        l_run[rt] *= alpha, z_run[rt] *= alpha;
        bsum[rt] *= alpha;
#pragma unroll
        for (int d = 0; d < D_TILES; ++d) acc[rt][d] *= alpha;
        m_run[rt] = m_new, neg_mc[rt] = neg;
      }
      float bv[8], z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) bv[e] = word_step(L.vw[e]), z[e] = word_offset(L.vw[e]);
      if (need_mask) {  // a key that a row does not read may hold anything, a NaN among it
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          bv[e] = (hidden >> e) & 1 ? 0.f : bv[e];
          z[e] = (hidden >> e) & 1 ? 0.f : z[e];
        }
      }
      float z_even = z_run[rt], z_odd = 0.f, l_even = l_run[rt], l_odd = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(x[e], scale_log2e, neg_mc[rt])), p1 = __builtin_amdgcn_exp2f(fmaf(x[e + 1], scale_log2e, neg_mc[rt]));
        l_even += p0, l_odd += p1;
        z_even = fmaf(p0, z[e], z_even), z_odd = fmaf(p1, z[e + 1], z_odd);
        bv[e] *= p0, bv[e + 1] *= p1;
      }
      l_run[rt] = l_even + l_odd, z_run[rt] = z_even + z_odd;
      if constexpr (EXACT) {
        Frag8 part[3];
        three_parts(bv, part);
        bf[rt][0] = part[0], bf[rt][1] = part[1], bf[rt][2 % B_PARTS] = part[2];
      } else {
        bf[rt][0].u = make_uint4(pack2_bf16(bv[0], bv[1]), pack2_bf16(bv[2], bv[3]), pack2_bf16(bv[4], bv[5]), pack2_bf16(bv[6], bv[7]));
        uint32_t rest[4];
        const uint32_t whole[4] = {bf[rt][0].u.x, bf[rt][0].u.y, bf[rt][0].u.z, bf[rt][0].u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          rest[i] = pack2_bf16(bv[2 * i] - __uint_as_float(whole[i] << 16), bv[2 * i + 1] - __uint_as_float(whole[i] & 0xffff0000u));
        bf[rt][1].u = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        bsum[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, bf[rt][1].v, bsum[rt], 0, 0, 0);
        bsum[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, bf[rt][0].v, bsum[rt], 0, 0, 0);
      }
    }
    // tile d of the output: 4 bits: dimension 64 c + 4 m + i of d = 4 c + i (the last two, where 32 are left, 64 c + 2 m + i);
    // 8 bits: 32 c + 2 m + i of d = 2 c + i
#pragma unroll
    for (int d = 0; d < D_TILES; ++d) {
      Frag8 vf;
      if constexpr (BITS == 4) {
        const uint32_t c0 = L.vc[2 * (d / 2)] >> (4 * (d & 1)), c1 = L.vc[2 * (d / 2) + 1] >> (4 * (d & 1));
        vf.u = make_uint4(codes.nibbles(c0), codes.nibbles(c0 >> 8), codes.nibbles(c1), codes.nibbles(c1 >> 8));
      } else {
        const uint32_t c0 = L.vc[(2 * d) % Keys::VC], c1 = L.vc[(2 * d + 1) % Keys::VC];
        vf.u = make_uint4(codes.bytes(c0, 0), codes.bytes(c0, 2), codes.bytes(c1, 0), codes.bytes(c1, 2));
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int p = B_PARTS - 1; p >= 0; --p) acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.v, bf[rt][p].v, acc[rt][d], 0, 0, 0);
    }
  };

  // The registers of BUFFERS tiles in turn, the loads of the tile BUFFERS - 1 on ahead of this one's arithmetic (a copy from one to
  // the other would wait for the loads).  A tile past the last one reads page 0's first keys where it is not a load of nothing.
  int tile = SPLIT ? wave : 0;
  if (tile < tiles) {
    Keys held[BUFFERS];
    page_ahead = look_up(32 * (tile0 + tile));
    if constexpr (!PAGE32) k_ahead = entry_of(32 * (tile0 + tile) + krel), v_ahead = entry_of(32 * (tile0 + tile) + 8 * j);
#pragma unroll
    for (int u = 0; u < BUFFERS - 1; ++u) issue(held[u], tile + u * STEP);
    for (bool more = true; more;) {
#pragma unroll
      for (int u = 0; u < BUFFERS; ++u) {
        issue(held[(u + BUFFERS - 1) % BUFFERS], tile + (BUFFERS - 1) * STEP);
        compute(held[u], 32 * (tile0 + tile));
        tile += STEP;
        if (tile >= tiles) {
          more = false;
          break;
        }
      }
    }
  }

  // ---- a row's sums over its lanes, and the output that the sums stand for ------------------- //
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l_run[rt] += __shfl_xor(l_run[rt], 16, 64);
    l_run[rt] += __shfl_xor(l_run[rt], 32, 64);
    z_run[rt] += __shfl_xor(z_run[rt], 16, 64);
    z_run[rt] += __shfl_xor(z_run[rt], 32, 64);
    const float add = fmaf(-C::OFF, bsum[rt][0], z_run[rt]);
#pragma unroll
    for (int d = 0; d < D_TILES; ++d) acc[rt][d] += add;
  }
  // calls put(first dimension, values) for the lane's share of a row: four values of neighbouring dimensions, or two
  auto each_piece = [&](int rt, auto&& put) {
    constexpr int FOURS = BITS == 4 ? G / 2 : 0;
#pragma unroll
    for (int c = 0; c < FOURS; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        put(64 * c + 16 * j + 4 * i, 4, (float4v){acc[rt][4 * c][i], acc[rt][(4 * c + 1) % D_TILES][i], acc[rt][(4 * c + 2) % D_TILES][i], acc[rt][(4 * c + 3) % D_TILES][i]});
#pragma unroll
    for (int d = 4 * FOURS; d < D_TILES; d += 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) put(16 * d + 8 * j + 2 * i, 2, (float4v){acc[rt][d][i], acc[rt][(d + 1) % D_TILES][i], 0.f, 0.f});
  };
  auto store_out = [&](T* row, int d, int count, float4v v) {
    if constexpr (EXACT) {
      *(float2*)(row + d) = make_float2(v[0], v[1]);
      if (count == 4) *(float2*)(row + d + 2) = make_float2(v[2], v[3]);
    } else {
      if (count == 4)
        *(uint2*)(row + d) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
      else
        *(uint32_t*)(row + d) = pack2_bf16(v[0], v[1]);
    }
  };

  if constexpr (!SPLIT) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (!row_valid[rt]) continue;
      if (slot < 0) {
        const float inv = page_missing ? not_a_number() : 1.0f / l_run[rt];
        T* row = out + (size_t)(q0 + ti[rt]) * out_stride + (size_t)hq[rt] * HEAD_DIM;
        each_piece(rt, [&](int d, int count, float4v v) { store_out(row, d, count, v * inv); });
      } else {
        // row tile k of a cut item has the slots from slot + k * (chunks of the item) on
        float* row = partial + (((size_t)slot + (size_t)(RT * wave + rt) * n_chunks) * n_kv_heads + g0) * 16 * PARTIAL_STRIDE + (size_t)n * PARTIAL_STRIDE;
        each_piece(rt, [&](int d, int count, float4v v) {
          *(float2*)(row + d) = make_float2(v[0], v[1]);
          if (count == 4) *(float2*)(row + d + 2) = make_float2(v[2], v[3]);
        });
        if (j == 0) {
          row[HEAD_DIM] = m_run[rt] * scale_log2e;
          row[HEAD_DIM + 1] = page_missing ? not_a_number() : l_run[rt];
        }
      }
    }
  } else {
    static_assert(!SPLIT || RT == 1, "a team shares one row tile");
    // the team's wavefronts join: the largest reference, every wavefront's sums and output scaled to it
    __shared__ float team_m[TEAM][16], team_l[TEAM][16];
    __shared__ __attribute__((aligned(16))) float team_o[TEAM][16][HEAD_DIM + 4];
    if (j == 0) {
      team_m[wave][n] = m_run[0];
      team_l[wave][n] = l_run[0];
    }
    __syncthreads();
    float m_all = neg_inf;
#pragma unroll
    for (int w2 = 0; w2 < TEAM; ++w2) m_all = fmaxf(m_all, team_m[w2][n]);
    float l_all = 0.f, mine = 0.f;
#pragma unroll
    for (int w2 = 0; w2 < TEAM; ++w2) {
      // -inf: that wavefront had no tile, or none with a key of this row, and sums of zeros; or all scores were NaN, and so are the
      // sums, which a factor of 0 leaves as they are
      const float mw = team_m[w2][n];
      const float f = mw == neg_inf ? 0.f : __builtin_amdgcn_exp2f((mw - m_all) * scale_log2e);
      l_all += team_l[w2][n] * f;
      if (w2 == wave) mine = f;
    }
    each_piece(0, [&](int d, int count, float4v v) {
      float* o = &team_o[wave][n][d];
      if (count == 4)
        *(float4v*)o = v * mine;
      else
        *(float2*)o = make_float2(v[0] * mine, v[1] * mine);
    });
    __syncthreads();
    if (!row_valid[0]) return;
    const float inv = page_missing ? not_a_number() : 1.0f / l_all;
    T* orow = out + (size_t)(q0 + ti[0]) * out_stride + (size_t)hq[0] * HEAD_DIM;
    float* prow = partial + (((size_t)max(slot, 0) * n_kv_heads + g0) * 16 + n) * PARTIAL_STRIDE;
    for (int d = 16 * wave + 4 * j; d < HEAD_DIM; d += 16 * TEAM) {
      float4v sum = *(const float4v*)&team_o[0][n][d];
#pragma unroll
      for (int w2 = 1; w2 < TEAM; ++w2) sum += *(const float4v*)&team_o[w2][n][d];
      if (slot < 0)
        store_out(orow, d, 4, sum * inv);
      else
        *(float4v*)(prow + d) = sum;
    }
    if (slot >= 0 && wave == 0 && j == 0) {
      prow[HEAD_DIM] = m_all * scale_log2e;
      prow[HEAD_DIM + 1] = page_missing ? not_a_number() : l_all;
    }
  }
}

// Joins the partial results of a row: merge item {sequence, first row, first slot, number of partials}; grid (items,
// key/value heads, 16 rows).  Wavefront w takes partials w, w + MERGE_WAVES, ..., four loads of each at a time.
#define MERGE_WAVES 4
template <typename T>
__global__ void __launch_bounds__(64 * MERGE_WAVES)
attention_quant_merge_kernel(T* __restrict__ out, long out_stride, const float* __restrict__ partial, const int* __restrict__ cu_q,
                             const int* __restrict__ merge, int n_q_heads, int n_kv_heads) {
  const int* item = merge + (size_t)blockIdx.x * 4;
  const int b = item[0], first = item[2], count = item[3];
  const int g = blockIdx.y, n = blockIdx.z, group = n_q_heads / n_kv_heads;
  const int q0 = cu_q[b], r = item[1] + n;
  if (r >= (cu_q[b + 1] - q0) * group || count <= 0) return;  // also null items, whose first row lies beyond every sequence's
  constexpr int PER = (HEAD_DIM + 63) / 64;
  const float neg_inf = -__builtin_inff();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ float top_of[MERGE_WAVES], l_of[MERGE_WAVES], o_of[MERGE_WAVES][HEAD_DIM];
  const float* rows = partial + (((size_t)first * n_kv_heads + g) * 16 + n) * PARTIAL_STRIDE;
  const size_t stride = (size_t)n_kv_heads * 16 * PARTIAL_STRIDE;
  float top = neg_inf;
  for (int p = threadIdx.x; p < count; p += 64 * MERGE_WAVES) top = fmaxf(top, rows[p * stride + HEAD_DIM]);
  top = wave_max(top);
  if (lane == 0) top_of[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < MERGE_WAVES; ++w) top = fmaxf(top, top_of[w]);
  float o[PER] = {}, l = 0.f;
  for (int p0 = wave; p0 < count; p0 += 4 * MERGE_WAVES) {
    float m[4], lp[4], op[4][PER];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* row = rows + min(p0 + u * MERGE_WAVES, count - 1) * stride;
      m[u] = row[HEAD_DIM], lp[u] = row[HEAD_DIM + 1];
#pragma unroll
      for (int i = 0; i < PER; ++i) op[u][i] = row[min(lane + 64 * i, HEAD_DIM - 1)];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p0 + u * MERGE_WAVES >= count) break;  // past the last partial
      // -inf: a chunk with no key of this row, whose sums are zeros, or one whose scores were all NaN, which stays
      const float f = m[u] == neg_inf ? 0.f : __builtin_amdgcn_exp2f(m[u] - top);
      l += f * lp[u];
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += f * op[u][i];
    }
  }
  if (lane == 0) l_of[wave] = l;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < HEAD_DIM) o_of[wave][lane + 64 * i] = o[i];
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < MERGE_WAVES; ++w) total += l_of[w];
  const int ti = r / group, d = threadIdx.x;
  if (d >= HEAD_DIM) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < MERGE_WAVES; ++w) sum += o_of[w][d];
  Elem<T>::store(out + (size_t)(q0 + ti) * out_stride + (size_t)(g * group + r - ti * group) * HEAD_DIM + d, sum / total);
}

extern "C" int cwm_attention_quant(const void* q, long q_stride, int dtype, void* out, long out_stride, const void* cache, const int* block_table,
                                   int table_width, const int* cu_q, const int* kv_len, const int* work, int n_work, const int* work_wide,
                                   int n_work_wide, int wide_tiles, const int* merge, int n_merge, float* partial, int n_q_heads, int n_kv_heads,
                                   int head_dim, int page_size, int num_pages, int window_left, float scale, int bits, hipStream_t stream) {
  QUANT_REQUIRE_SIZES("attention_quant");
  CWM_REQUIRE(head_dim == HEAD_DIM, "attention_quant: this library is built for head_dim %d, not %d", HEAD_DIM, head_dim);
  CWM_REQUIRE(n_q_heads > 0 && n_q_heads % n_kv_heads == 0, "attention_quant: %d query heads do not divide into %d key/value heads", n_q_heads, n_kv_heads);
  const int piece = dtype == CWM_BF16 ? 8 : 4;
  CWM_REQUIRE(q_stride % piece == 0 && out_stride % 4 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)cache % 16 == 0,
              "attention_quant: rows must be 16-byte aligned");
  CWM_REQUIRE(n_work >= 0 && n_work_wide >= 0 && n_merge >= 0, "attention_quant: negative work counts");
  CWM_REQUIRE(n_work_wide == 0 || wide_tiles == 8, "attention_quant: wide items have 8 row tiles, not %d", wide_tiles);
  CWM_REQUIRE(n_merge == 0 || partial, "attention_quant: partial buffer missing");
  CWM_REQUIRE(scale > 0.f, "attention_quant: the scale is positive");
  CWM_REQUIRE((unsigned long long)quant_token_bytes(head_dim, bits) * page_size < (1ull << 31), "attention_quant: a page of %d keys is too large", page_size);
  CWM_REQUIRE(n_kv_heads <= 65535 && (long long)(n_work + n_work_wide) * n_kv_heads <= 0x7fffffffLL, "attention_quant: too much work");
  const float scale_log2e = scale * 1.4426950408889634f;
  int page_shift = -1;
  if ((page_size & (page_size - 1)) == 0) {
    page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
  }
#define CALL_ATTEND(T, BITS, RT, SPLIT, PAGE32, WORK, COUNT)                                                                                        \
  hipLaunchKernelGGL((attention_quant_kernel<T, BITS, RT, SPLIT, PAGE32>), dim3((unsigned)((COUNT)*n_kv_heads)), dim3(256), 0, stream, (const T*)q, \
                     q_stride, (T*)out, out_stride, (const uint8_t*)cache, block_table, table_width, cu_q, kv_len, WORK, partial, n_q_heads,        \
                     n_kv_heads, page_size, page_shift, num_pages, window_left, scale_log2e)
#define CALL_BITS(T, RT, SPLIT, PAGE32, WORK, COUNT) \
  if (bits == 4)                                     \
    CALL_ATTEND(T, 4, RT, SPLIT, PAGE32, WORK, COUNT); \
  else                                               \
    CALL_ATTEND(T, 8, RT, SPLIT, PAGE32, WORK, COUNT)
#define CALL_PAGES(T, RT, SPLIT, WORK, COUNT)      \
  if (page_size % 32 == 0) {                       \
    CALL_BITS(T, RT, SPLIT, true, WORK, COUNT);    \
  } else {                                         \
    CALL_BITS(T, RT, SPLIT, false, WORK, COUNT);   \
  }
  if (n_work > 0) {
    if (dtype == CWM_BF16) {
      CALL_PAGES(bf16_t, 1, true, work, n_work)
    } else {
      CALL_PAGES(float, 1, true, work, n_work)
    }
    if (int status = cwm_launch_status("attention_quant")) return status;
  }
  if (n_work_wide > 0) {
    CWM_REQUIRE(dtype == CWM_F32, "attention_quant: bfloat16 portions of many rows read unpacked keys and values");
    CALL_PAGES(float, 2, false, work_wide, n_work_wide)
    if (int status = cwm_launch_status("attention_quant (rows)")) return status;
  }
  if (n_merge > 0) {
    const dim3 grid(n_merge, n_kv_heads, 16), block(64 * MERGE_WAVES);
    if (dtype == CWM_BF16)
      hipLaunchKernelGGL((attention_quant_merge_kernel<bf16_t>), grid, block, 0, stream, (bf16_t*)out, out_stride, partial, cu_q, merge, n_q_heads, n_kv_heads);
    else
      hipLaunchKernelGGL((attention_quant_merge_kernel<float>), grid, block, 0, stream, (float*)out, out_stride, partial, cu_q, merge, n_q_heads, n_kv_heads);
    if (int status = cwm_launch_status("attention_quant (merge)")) return status;
  }
  return 0;
}
