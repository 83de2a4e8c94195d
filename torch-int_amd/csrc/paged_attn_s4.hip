// Causal attention of a batch's new tokens over a paged cache in 4 bits, all of it or a window of the last keys and some first ones:
//   ctx = alpha_pv * sum_j 2^(c x_j - M) v_j / sum_j 2^(c x_j - M),   x_j = q . k_j,  c = alpha_qk log2(e),
// over the positions j <= p that the token at p sees: p - j < window, or j < sinks.
// Keys and values are step (u - z), exact in fp16, and so are queries of int8 and fp16 (bf16 ones are rounded where they lie outside
// fp16's normal range): products of both kinds are fp16 MFMA with fp32 sums.  One pass over the keys with a running reference M.
//
// Work items, rows and slices as in the attention over the int8 cache (paged_items.h).  Keys that no row of an item sees are left out:
// an item counts the blocks of 16 keys with first ones in them, then those of its rows' windows, as one run of places.
#include "paged_items.h"

namespace ti {

// A nibble in the low bits of a 16-bit half, or in the next four, is a number of fp16 with one bit operation: 0x6400 + u is 1024 + u,
// 0x5400 + 16 u is 64 + u.  Less the same with z, times the step: exact.  `c` has two bytes in each half (of two columns, or of two
// keys); the four results are the low byte's nibbles, then the high byte's.
struct S4Bits {
  unsigned low_mask, high_mask, low_one, high_one;
  // masks in scalar registers, exponents in vector ones: one v_and_or_b32, which takes no constants of 32 bits, is enough then
  __device__ __forceinline__ S4Bits() : low_mask(0x000f000fu), high_mask(0x00f000f0u), low_one(0x64006400u), high_one(0x54005400u) {
    asm("" : "+s"(low_mask), "+s"(high_mask), "+v"(low_one), "+v"(high_one));
  }
  __device__ __forceinline__ unsigned low(unsigned c) const { return (c & low_mask) | low_one; }
  __device__ __forceinline__ unsigned high(unsigned c) const { return (c & high_mask) | high_one; }
};
// The same without the step: u - z.
struct S4Zero {
  v2h base[2];
  __device__ __forceinline__ void set(const S4Bits& b, int nibble, unsigned word) {
    base[nibble] = __builtin_bit_cast(v2h, b.low(word));
    if (nibble) base[nibble] -= v2h{(_Float16)960.0f, (_Float16)960.0f};
  }
  __device__ __forceinline__ v2h code(const S4Bits& b, unsigned c, int nibble) const {
    return __builtin_bit_cast(v2h, nibble ? b.high(c) : b.low(c)) - base[nibble];
  }
  __device__ __forceinline__ void codes(const S4Bits& b, unsigned c, v2h (&y)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = code(b, i >> 1 ? c >> 8 : c, i & 1);
  }
};
struct S4Two {
  v2h step[2], base[2];  // of low nibbles and of high ones: the step, and 1024 + z or 64 + z
  __device__ __forceinline__ void set(const S4Bits& b, int nibble, unsigned word) {  // `word`: a word in each half
    const unsigned s = word & 0x7ff07ff0u, z = b.low(word);
    step[nibble] = __builtin_bit_cast(v2h, s);
    base[nibble] = __builtin_bit_cast(v2h, z);
    if (nibble) base[nibble] -= v2h{(_Float16)960.0f, (_Float16)960.0f};
  }
  __device__ __forceinline__ void values(const S4Bits& b, unsigned c, v2h (&y)[4]) const {
    const unsigned d = c >> 8;
    const unsigned w[4] = {b.low(c), b.high(c), b.low(d), b.high(d)};
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (__builtin_bit_cast(v2h, w[i]) - base[i & 1]) * step[i & 1];
  }
};

__device__ __forceinline__ v8h join8(v2h a, v2h b, v2h c, v2h d) {
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

typedef unsigned short v2us __attribute__((ext_vector_type(2)));

// The sum over the four lanes n, n + 16, n + 32, n + 48, in all of them.
__device__ __forceinline__ float rows_add(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// The largest of all lanes, the same in all.
__device__ __forceinline__ unsigned wave_max(unsigned x) {
  auto step = [&](auto ctrl, auto rows) {
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    x = x > y ? x : y;
  };
  step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
  step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// Eight neighbouring elements of a query as fp16, in the order 0 2 1 3 4 6 5 7 in which the nibbles of two dwords come apart.
__device__ __forceinline__ v8h query8(const void* q, int type, long long at) {
  unsigned w[4];
  if (type == PT_S8) {
    const int2 x = *reinterpret_cast<const int2*>(static_cast<const int8_t*>(q) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // bytes plus 128 are the low bits of 1024 + them
      const unsigned u = ((unsigned)(i < 2 ? x.x : x.y) ^ 0x80808080u) >> (8 * (i & 1)) & 0x00ff00ffu;
      const v2h y = __builtin_bit_cast(v2h, u | 0x64006400u) - v2h{(_Float16)1152.0f, (_Float16)1152.0f};
      w[i] = __builtin_bit_cast(unsigned, y);
    }
  } else {
    const v4i x = *reinterpret_cast<const v4i*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(x[i | 1], x[i & 2], i & 1 ? 0x07060302u : 0x05040100u);
    if (type == PT_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2f y = {__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)};
        w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(y, v2h));
      }
    }
    // an infinity becomes NaN: scores of minus infinity alone would make a row that has seen no key
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v2h y = __builtin_bit_cast(v2h, w[i]);
      w[i] = __builtin_bit_cast(unsigned, y + (y - y));
    }
  }
  return join8(__builtin_bit_cast(v2h, w[0]), __builtin_bit_cast(v2h, w[1]), __builtin_bit_cast(v2h, w[2]), __builtin_bit_cast(v2h, w[3]));
}

// The keys that an item reads, as one run of places: `shift` keys are left out behind the first `head`.
struct S4Span {
  int keys;   // of the item's last row, as positions
  int head;   // places of first keys, a multiple of 16
  int shift;  // a multiple of 16
  __device__ __forceinline__ S4Span(const PagedAttn4& a, int first_position, int last_position) {
    keys = last_position < 0 ? 0 : last_position + 1;
    head = shift = 0;
    if (a.window > 0 && first_position >= a.window) {
      const int from = (first_position - a.window + 1) & ~15, first = (a.sinks + 15) & ~15;
      head = first < from ? first : from;
      shift = from - head;
    }
  }
  __device__ __forceinline__ int places() const { return keys - shift; }
  __device__ __forceinline__ int key(int place) const { return place < head ? place : place + shift; }
};

// Few rows: 16 to a workgroup, its four waves take 32 keys each in turn.  A SIMD issues one instruction of any kind in four cycles, and
// with one or a few rows to a key that is what bounds it, so what is done to a code is as little as can be: it becomes u - z, and
// the steps are multiplied into scores and weights:
//   q . k = s sum q (u - z),   sum_j p_j v_j = sum_j (p_j s_j) (u_j - z_j),
// where the weights p s go in as two fp16 numbers (22 bits).  Two groups have sums and weights of their own.  Steps reach from 2^-20
// to 2^13, so the reference M keeps p times the largest step of the keys so far at 2^15 or less, and the row's largest p times it at 2^8 or
// more.  The second fp16 number ends at 2^-24, so p is off by 2^-32 of the largest p times the largest step over its own at most: more
// than 22 bits' worth where a heavy key's step is 2^-10 of the largest or less.
// (Codes as they are, subnormal fp16 numbers u 2^-24, and z times the sums of q and of weights taken off behind the products
// would be a fifth less to issue, but the matrix pipe adds subnormal numbers with 2^-20 of their sum lost.)
// One token to each of 28 sequences of 1500 keys, 40 heads of 128: 39 us, 3.4 TB/s; 75 of up to 7003, 32 heads on 8: 75 us, 3.9 TB/s;
// one of 200000, 64 heads on 8: 57 us, 3.8 TB/s.  40 % of the issue slots of a 32-key step are codes becoming numbers (2.25 instructions
// to two), a third scores, steps and weights, a sixth addresses; half of the waves that fit are there on average, as workgroups begin
// (item, table, addresses, first keys: 5 us) and end.
constexpr int S4_HELD = 4;  // times 64 sequences
constexpr int s4_rows_lds(int DP) { return PA_WAVES * PA_ROWS * (DP + 4 + 2) * 4; }
template <int DP, int GROUPS, int OUT>
__device__ __forceinline__ void s4_rows(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const PagedPlan& p, int index,
                                        char* lds) {
  constexpr int NB = DP / 16;  // column blocks; lane n of 16 has NB / 2 bytes of a value row, from NB / 2 * n on
  constexpr int KW = DP / 32;  // dwords of a key row that a lane has
  const auto sum = reinterpret_cast<float(*)[PA_ROWS][DP + 4]>(lds);
  const auto offs = reinterpret_cast<float(*)[PA_ROWS]>(lds + PA_WAVES * PA_ROWS * (DP + 4) * 4);
  const auto den = offs + PA_WAVES;

  const PagedItem it = paged_item<4, false, true, S4_HELD>(b, c.page_shift, c.heads, PA_ROWS, p, index);
  if (!it.found) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int G = p.group, live_rows = it.s.T * G, half = c.D / 2;
  const int row = it.tile * PA_ROWS + n;  // of this lane's scores
  const int t = row / G, g = row - t * G;
  const int base = it.s.len - it.s.T;     // position of the first new token (negative: it has none)
  const bool real = row < live_rows;
  // the row sees positions below `limit`, from `from` on or below `sinks`; rows that nobody asked for see what they like
  const int limit = real ? base + t + 1 : 0x7fffffff;
  const int from = real && a.window > 0 ? limit - a.window : -0x7fffffff;
  int last_row = it.tile * PA_ROWS + PA_ROWS - 1;
  last_row = last_row < live_rows - 1 ? last_row : live_rows - 1;
  const int p0 = base + it.tile * PA_ROWS / G, p1 = base + last_row / G;  // positions of the first row and of the last one
  const S4Span span(a, p0, p1);
  const int places = span.places();
  const int all_from = a.window > 0 ? p1 + 1 - a.window : -0x7fffffff;  // from here on the last row sees the keys, and so do the others
  const int any_from = a.window > 0 ? p0 + 1 - a.window : -0x7fffffff;  // before it no row does, but for first ones
  const long long lo_ll = (long long)it.split * it.slice;
  const int lo = lo_ll < places ? (int)lo_ll : places;
  const int hi = lo_ll + it.slice < places ? (int)(lo_ll + it.slice) : places;

  // A lane has the bytes KW * 4 * kg .. of a key row, and what the row's end has no such bytes for, the last ones before it, where Q is zero.
  const int kbyte = kg * KW * 4 <= half - KW * 4 ? kg * KW * 4 : half - KW * 4;
  v8h qf[KW];  // of low nibbles, then of high ones
  {
    const long long from_q = (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head;
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const int byte = kbyte + i % (KW / 2) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[i][j] = (_Float16)0.0f;
      if (real && byte >= kg * KW * 4 && byte < half) qf[i] = query8(a.q, a.q_type, from_q + byte + (i < KW / 2 ? 0 : half));
    }
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const uint8_t* kb = c.k + it.head * c.head;
  const uint8_t* vb = c.v + it.head * c.head;
  const char* ksb = reinterpret_cast<const char*>(c.k_scale) + it.head * c.scale_head;
  const char* vsb = reinterpret_cast<const char*>(c.v_scale) + it.head * c.scale_head;
  const int* const table = b.table + (long long)it.seq * b.per_seq;
  const int mask = (1 << c.page_shift) - 1, last_block = hi > 0 ? (hi - 1) >> 4 : 0;
  const int head_blocks = span.head >> 4, shift_blocks = span.shift >> 4;

  float off = PA_EMPTY, dsum = 0.0f, most = 35.0f;  // 2^most times the largest step so far is 2^15 (the smallest there is: 2^-20)
  unsigned top_word = 15;                           // a word no less than those so far, bits of z set
  v4f acc[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = v4f{0, 0, 0, 0};

  // The places of the wave's next 64 blocks of 16 keys, two to a step, one to a lane: bytes from a pool's start, first key, and whether
  // there is something to hide in it.  Blocks behind the last key are hidden, and read where there is memory.
  constexpr int STRIDE = PA_WAVES * 32;
  unsigned long long code = 0, word = 0, odd = 0, lost = 0;
  int key = 0;
  auto look = [&](int s0) {
    const int place = (s0 >> 4) + (lane >> 1) * (STRIDE / 16) + (lane & 1);
    int at = place < last_block ? place : last_block;
    at = at < head_blocks ? at : at + shift_blocks;
    key = at << 4;
    const int page = table[key >> c.page_shift];
    const bool have = (unsigned)page < (unsigned)c.pages;
    const unsigned long long there = have ? (unsigned)page : 0u;
    code = there * c.page + (unsigned)((key & mask) * c.token);
    word = there * c.scale_page + (unsigned)((key & mask) * (2 * GROUPS));
    lost = __ballot(!have);
    odd = lost | __ballot((place << 4) + 16 > hi || key + 16 > p0 + 1 || key < all_from);
  };
  // by buffer instructions: what a lane adds is one register, the block's place in scalar ones
  auto pool = [](const void* from) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, -1, 0x00020000); };
  auto lane64 = [](unsigned long long x, int i) {
    return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, i);
  };
  const unsigned kcol = (unsigned)(n * c.token) + (unsigned)kbyte;
  const int vbyte = (n * NB / 2) & ~3;
  const unsigned vcol = (unsigned)(kg * 4 * c.token) + (vbyte < half ? (unsigned)vbyte : 0u);
  int k[2][KW];
  unsigned v[8], kz[2], ks[2][2 * GROUPS], vs[2][2 * GROUPS];  // (words of K: of the lane's key, and of those whose scores it gets)
  auto fetch_words = [&](unsigned (&w)[2 * GROUPS], const char* from) {
    const auto r = pool(from);
    if constexpr (GROUPS == 2) {
      const v4i x = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, kg * 16, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (unsigned)x[i];
    } else {
      const int2 x = __builtin_bit_cast(int2, __builtin_amdgcn_raw_buffer_load_b64(r, kg * 8, 0, 0));
      w[0] = (unsigned)x.x, w[1] = (unsigned)x.y;
    }
  };
  struct Places {
    unsigned long long code[2], word[2];
  };
  auto places_of = [&](int i) {  // of step i of the 32 that have been looked up
    Places w;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) w.code[blk] = lane64(code, 2 * i + blk), w.word[blk] = lane64(word, 2 * i + blk);
    return w;
  };
  auto fetch_k = [&](const Places& w) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const auto r = pool(kb + w.code[blk]);
      if constexpr (KW == 4) {
        const v4i x = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, kcol, 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) k[blk][i] = x[i];
      } else {
        const int2 x = __builtin_bit_cast(int2, __builtin_amdgcn_raw_buffer_load_b64(r, kcol, 0, 0));
        k[blk][0] = x.x, k[blk][1] = x.y;
      }
      fetch_words(ks[blk], ksb + w.word[blk]);
      if constexpr (GROUPS == 2) kz[blk] = __builtin_amdgcn_raw_buffer_load_b32(pool(ksb + w.word[blk]), n * 4, 0, 0);
      else kz[blk] = __builtin_amdgcn_raw_buffer_load_b16(pool(ksb + w.word[blk]), n * 2, 0, 0);
    }
  };
  auto fetch_v = [&](const Places& w) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      fetch_words(vs[blk], vsb + w.word[blk]);
      const auto r = pool(vb + w.code[blk]);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[blk * 4 + j] = __builtin_amdgcn_raw_buffer_load_b32(r, vcol, j * c.token, 0);
    }
  };
  const S4Bits bits;
  unsigned steps = 0x7ff07ff0u;
  float minus = -1.0f;  // (kept out of the compiler's sight, as the zero is put in its way, for one instruction instead of two)
  asm("" : "+s"(steps), "+v"(minus));
  auto halves = [](unsigned x) { return __builtin_bit_cast(v2h, x); };
  auto times = [](_Float16 s, float x) { return __builtin_fmaf((float)s, x, 0.0f); };
  auto scores = [&](float (&x)[8]) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      S4Zero zero;
      zero.set(bits, 0, __builtin_amdgcn_perm(kz[blk], kz[blk], 0x01000100u));
      zero.set(bits, 1, __builtin_amdgcn_perm(kz[blk], kz[blk], GROUPS == 2 ? 0x03020302u : 0x01000100u));
      v4f d0 = {0, 0, 0, 0}, d1 = {0, 0, 0, 0};  // of low nibbles and of high ones
#pragma unroll
      for (int i = 0; i < KW / 2; ++i) {
        v2h u[4], w[4];
        zero.codes(bits, (unsigned)k[blk][2 * i], u);
        zero.codes(bits, (unsigned)k[blk][2 * i + 1], w);
        d0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(u[0], u[2], w[0], w[2]), qf[i], d0, 0, 0, 0);
        v4f& high = GROUPS == 2 ? d1 : d0;
        high = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(u[1], u[3], w[1], w[3]), qf[KW / 2 + i], high, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (GROUPS == 2) {
          const v2h s = halves(ks[blk][r] & steps);
          x[blk * 4 + r] = __builtin_fmaf((float)s[0], d0[r], times(s[1], d1[r]));
        } else {
          x[blk * 4 + r] = times(halves(ks[blk][r >> 1] & steps)[r & 1], d0[r]);
        }
      }
    }
  };
  const unsigned vpick = DP == 128 || (n & 1) == 0 ? 0x05040100u : 0x07060302u;  // the half of a dword of V that this lane has
  auto work = [&](float (&x)[8], int s0, int i0) {
    if (odd >> (2 * i0) & 3) {
      // What no row sees is not there: its values' steps, which may be anything, become zeros.
      const int key0 = __builtin_amdgcn_readlane(key, 2 * i0), key1 = __builtin_amdgcn_readlane(key, 2 * i0 + 1);
      const bool gone[2] = {(lost >> (2 * i0) & 1) != 0, (lost >> (2 * i0) & 2) != 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int mine = (i >> 2 ? key1 : key0) + kg * 4 + (i & 3);
        const bool dead = s0 + (i >> 2) * 16 + kg * 4 + (i & 3) >= hi || gone[i >> 2] || (mine < any_from && mine >= a.sinks);
        if (dead || mine >= limit || (mine < from && mine >= a.sinks)) x[i] = -__builtin_inff();
        if (GROUPS == 2) {
          if (dead) vs[i >> 2][i & 3] = 0;
        } else if (dead) {
          vs[i >> 2][(i & 3) >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
        }
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
    // the largest word of the lane's, both halves; where one is larger than all before, p has to be less
    v2us larger = __builtin_bit_cast(v2us, vs[0][0]);
#pragma unroll
    for (int i = 1; i < 4 * GROUPS; ++i) larger = __builtin_elementwise_max(larger, __builtin_bit_cast(v2us, vs[i / (2 * GROUPS)][i % (2 * GROUPS)]));
    const unsigned largest = larger[0] > larger[1] ? larger[0] : larger[1];
    if (__ballot(largest > top_word) != 0) {
      // (the top bit and those of z are no part of a step; the next power of two)
      const unsigned all = wave_max(largest) & 0x7fffu;
      top_word = top_word > (all | 0x3ff) ? top_word : all | 0x3ff;
      const int exponent = (int)(top_word >> 10) - 14;
      most = 15.0f - (float)(exponent < -20 ? -20 : exponent);
    }
    // a new reference only where a weight could pass 2^15: it starts at 2^8, fp16 ends at 2^16
    if (__ballot(__builtin_fmaf(top, cl, off) > most) != 0) {
      top = rows_max(top);
      if (__builtin_fmaf(top, cl, off) > most) {
        const float fresh = most - 7.0f - top * cl;
        const float scale = __builtin_amdgcn_exp2f(fresh - off);
        off = fresh;
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] *= scale;
        dsum *= scale;
      }
    }
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], cl, off));
      dsum += e[i];
    }
    // pairs of keys side by side, of a dword's lower half and its upper one
    unsigned pairs[NB / 4][4];
#pragma unroll
    for (int h = 0; h < NB / 4; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) pairs[h][j] = __builtin_amdgcn_perm(v[2 * j + 1], v[2 * j], h ? 0x07060302u : vpick);
    S4Zero zero[4];  // of the pairs
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      v2h hi2[4], lo2[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned both = vs[j >> 1][j & 1];
        if constexpr (GROUPS == 2)
          both = __builtin_amdgcn_perm(vs[j >> 1][2 * (j & 1) + 1], vs[j >> 1][2 * (j & 1)], q ? 0x07060302u : 0x05040100u);
        if (GROUPS == 2) zero[j].set(bits, q, both);
        else zero[j].set(bits, 0, both), zero[j].set(bits, 1, both);
        const v2h s = halves(both & steps);
        const v2f y = {times(s[0], e[2 * j]), times(s[1], e[2 * j + 1])};
        hi2[j] = __builtin_convertvector(y, v2h);
        const v2f rest = {__builtin_fmaf((float)hi2[j][0], minus, y[0]), __builtin_fmaf((float)hi2[j][1], minus, y[1])};
        lo2[j] = __builtin_convertvector(rest, v2h);
      }
      const v8h hi_w = join8(hi2[0], hi2[1], hi2[2], hi2[3]), lo_w = join8(lo2[0], lo2[1], lo2[2], lo2[3]);
#pragma unroll
      for (int h = 0; h < NB / 4; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (GROUPS == 2 && (i & 1) != q) continue;
          v2h y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = zero[j].code(bits, i >> 1 ? pairs[h][j] >> 8 : pairs[h][j], i & 1);
          const v8h vf = join8(y[0], y[1], y[2], y[3]);
          acc[4 * h + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, hi_w, acc[4 * h + i], 0, 0, 0);
          acc[4 * h + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, lo_w, acc[4 * h + i], 0, 0, 0);
        }
    }
  };

  // A step's keys are asked for as soon as those of the step before have become scores, its values when those have become sums.
  int s0 = lo + wave * 32;
  if (s0 < hi) {
    // Waits count loads, in the order in which they were issued: keys before values on every way into the loop, which the barriers keep
    // so, or the wait for keys would be one for the values behind them as well.
    look(s0);
    Places next = places_of(0);
    fetch_k(next);
    __builtin_amdgcn_sched_barrier(0);
    fetch_v(next);
    __builtin_amdgcn_sched_barrier(0);
    for (int i = 0;; ++i) {
      float x[8];
      scores(x);
      // (the places behind the 32nd step's are not known yet: its own again, which nobody uses)
      next = places_of(i + 1 < 32 ? i + 1 : 31);
      __builtin_amdgcn_sched_barrier(0);
      fetch_k(next);
      __builtin_amdgcn_sched_barrier(0);
      work(x, s0, i);
      __builtin_amdgcn_sched_barrier(0);
      fetch_v(next);
      __builtin_amdgcn_sched_barrier(0);
      s0 += STRIDE;
      if (s0 >= hi) break;
      if (i == 31) {
        look(s0);
        next = places_of(0);
        fetch_k(next);
        __builtin_amdgcn_sched_barrier(0);
        fetch_v(next);
        __builtin_amdgcn_sched_barrier(0);
        i = -1;
      }
    }
  }

  // The waves meet: acc[4 h + 2 i + nibble][r] of lane (n, kg) is row n's column 2 h + i of the NB / 2 from NB / 2 (4 kg + r) on, in
  // the half of the nibble.
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nib = 0; nib < 2; ++nib) {
      float* const to = &sum[wave][n][nib * (DP / 2) + NB / 2 * (4 * kg + r)];
      if constexpr (NB == 8) *reinterpret_cast<v4f*>(to) = v4f{acc[nib][r], acc[2 + nib][r], acc[4 + nib][r], acc[6 + nib][r]};
      else *reinterpret_cast<v2f*>(to) = v2f{acc[nib][r], acc[2 + nib][r]};
    }
  dsum = rows_add(dsum);
  if (kg == 0) {
    offs[wave][n] = off;
    den[wave][n] = dsum;
  }
  __syncthreads();
  const PagedOut to = {a.out, a.q_heads, c.D, a.alpha_pv};
  const PagedRows out_row(it, a.q_heads, G, PA_ROWS);
  for (int e = threadIdx.x; e < PA_ROWS * (DP / 4); e += PA_THREADS) {
    const int r = e / (DP / 4), d = (e % (DP / 4)) * 4, column = paged_column<DP>(d, c.D);
    const int rr = it.tile * PA_ROWS + r;
    if (rr >= live_rows || column >= c.D) continue;
    float least = offs[0][r];
#pragma unroll
    for (int w = 1; w < PA_WAVES; ++w) least = offs[w][r] < least ? offs[w][r] : least;
    float y[4] = {0, 0, 0, 0}, l = 0;
#pragma unroll
    for (int w = 0; w < PA_WAVES; ++w) {
      const float scale = __builtin_amdgcn_exp2f(least - offs[w][r]);
      const v4f v = *reinterpret_cast<const v4f*>(&sum[w][r][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i] * scale;
      l += den[w][r] * scale;
    }
    if (it.splits > 1) {
      const long long slot = it.place + (long long)it.split * it.step;
      put4(p.ws + (slot * PA_ROWS + r) * DP + d, y[0], y[1], y[2], y[3]);
      if (d == 0) put2(p.ws + (long long)p.places * PA_ROWS * DP + (slot * PA_ROWS + r) * 2, least, l);
    } else {
      const float f = l != 0.0f ? a.alpha_pv / l : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = l != 0.0f ? y[i] * f : 0.0f;
      store_some<4, OUT>(a.out, out_row(r) * c.D + column, y);
    }
  }
  if (it.splits > 1) meet_and_join<PA_ROWS, DP, OUT, true>(to, p, it, reinterpret_cast<int*>(&offs[0][0]), &sum[0][0][0]);
}

// Many rows: 128 to a workgroup, 32 to each of its four waves, 64 keys to a step.  Each wave brings 16 of a step's keys from memory, a
// step ahead of their becoming numbers, and writes them to the LDS as fp16: keys as rows, 16-byte chunks (eight bytes' low
// nibbles, or high ones) exchanged by the row; values in the order in which MFMA operands are read, of eight keys, chosen as
// S^T = K Q^T leaves them in a lane, one column in 16 bytes, lane after lane.  One unpacking then serves 128 rows.
// Column block i of V holds, of lane m's NDB / 2 bytes of a row, byte i / 2's low nibble or high one.
//
// A step is two halves of 32 keys with a barrier behind each.  The instructions of a half are laid out as bundles of one matrix
// instruction and what fits beside it: the scores of the next half and the sums of the one before are on their way while this one's
// become weights and the next step's codes numbers.  1536 rows over 12288 keys, 32 heads on 8: 448 us with one after the other, 397 so,
// 712 TFLOP/s.  Two workgroups to a CU fill the LDS and the registers; the matrix pipe is busy for 32 % of the clocks, the vector ALUs for 49, 8
// are LDS conflicts, and what bounds it is issue.
// A weight is one fp16 number, 11 bits: a second one would be 16 matrix instructions more to the 32 of a step.  A context is off by 2^-11 of
// sum w |v| / sum w at most, by far less where many keys count, as their errors are independent: against 64 bits, 3 x 700 tokens of normal
// values, 40 heads, fp16 out, by 0.00024 of its norm, of which rounding the output alone is 0.00021; bf16 out 0.0017 with and without.
// Where values cancel it can be more than the output's rounding, which is 2^-11 of what is left of them.
constexpr int ST_ROWS = 128, ST_KEYS = 64;
constexpr int ST_PARTS = 4;
constexpr int ST_JOIN = 32;      // rows that a workgroup joins
constexpr int ST_PLENTY = 2048;  // items from which on nothing is cut: four rounds, whose last one is a small part
constexpr int ST_AT_ONCE = 512;  // workgroups on the chip
constexpr int ST_TARGET = 1536;  // slices, at most about (1536 rows over 12288 keys 397 us; with 768 424, which is two rounds of 384 at best)
constexpr int s4_tiles_lds(int DP) { return 2 * 2 * ST_KEYS * DP * 2; }  // two steps of K, then of V
template <int DP, int GROUPS, int OUT>
__device__ __forceinline__ void s4_tiles(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const PagedPlan& p, int index,
                                         char* lds) {
  constexpr int NDB = DP / 32;  // column blocks of O^T
  constexpr int KS = DP / 16;   // steps of 16 along a key row
  constexpr int KW = DP / 32;   // dwords of a key row that a thread brings
  constexpr int BYTES = ST_KEYS * DP * 2;  // of a step of K, or of V

  const PagedItem it = paged_item<ST_PARTS, false, false, S4_HELD>(b, c.page_shift, c.heads, ST_ROWS, p, index);
  if (!it.found) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int G = p.group, live_rows = it.s.T * G, half = c.D / 2;
  const int base = it.s.len - it.s.T;
  const int row0 = it.tile * ST_ROWS + wave * 32, row = row0 + n;
  const int t = row / G, g = row - t * G;
  const bool real = row < live_rows;
  const int limit = real ? base + t + 1 : 0x7fffffff;
  const int from = real && a.window > 0 ? limit - a.window : -0x7fffffff;
  // positions of the workgroup's first and last rows, and of the wave's (one without rows: behind everything, it sees no key)
  const int last_row = it.tile * ST_ROWS + ST_ROWS - 1 < live_rows - 1 ? it.tile * ST_ROWS + ST_ROWS - 1 : live_rows - 1;
  const int p0 = base + it.tile * ST_ROWS / G, p1 = base + last_row / G;
  const int w0 = base + row0 / G, w1 = row0 < live_rows ? base + (row0 + 31 < live_rows ? row0 + 31 : live_rows - 1) / G : -1;
  const S4Span span(a, p0, p1);
  const int places = span.places();
  const int any_from = a.window > 0 ? p0 + 1 - a.window : -0x7fffffff;       // before it no row sees keys, but for first ones
  const int wave_all_from = a.window > 0 ? w1 + 1 - a.window : -0x7fffffff;  // from here on all of its rows do
  const long long lo_ll = (long long)it.split * it.slice;
  const int lo = lo_ll < places ? (int)lo_ll : places;
  const int hi = lo_ll + it.slice < places ? (int)(lo_ll + it.slice) : places;

  int keys = w1 + 1 - span.shift;  // places up to the wave's last key
  keys = keys < 0 ? 0 : keys < hi ? keys : hi;

  v8h qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int chunk = 2 * i + h, byte = chunk % (DP / 16) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) qf[i][j] = (_Float16)0.0f;
    if (real && byte < half)
      qf[i] = query8(a.q, a.q_type, (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head + byte +
                                        (chunk < DP / 16 ? 0 : half));
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const uint8_t* kb = c.k + it.head * c.head;
  const uint8_t* vb = c.v + it.head * c.head;
  const char* ksb = reinterpret_cast<const char*>(c.k_scale) + it.head * c.scale_head;
  const char* vsb = reinterpret_cast<const char*>(c.v_scale) + it.head * c.scale_head;
  const auto table = (const __attribute__((address_space(4))) int*)(b.table + (long long)it.seq * b.per_seq);
  const int mask = (1 << c.page_shift) - 1, last_block = hi > 0 ? (hi - 1) >> 4 : 0;
  const int head_blocks = span.head >> 4, shift_blocks = span.shift >> 4;
  const S4Bits bits;

  // the first key of a block of 16 places; blocks behind the last key are masked, and read where there is memory
  auto key_of = [&](int block) {
    int at = block < last_block ? block : last_block;
    at = at < head_blocks ? at : at + shift_blocks;
    return at << 4;
  };
  auto have = [&](int page) { return (unsigned)page < (unsigned)c.pages; };
  auto pool = [](const void* from) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, -1, 0x00020000); };

  // What this thread brings of a step: of the wave's 16 keys, KW dwords of K and the NDB / 2 bytes n NDB / 2 .. of eight rows of V.
  const int krow = lane >> 2;
  const int kbyte = (lane & 3) * KW * 4 <= half - KW * 4 ? (lane & 3) * KW * 4 : half - KW * 4;
  const unsigned kcol = (unsigned)(krow * c.token + kbyte);
  const int vbyte = n * (NDB / 2);
  const unsigned vcol = (unsigned)(h * 4 * c.token) + (vbyte < half ? (unsigned)vbyte : 0u);
  int kreg[KW];
  unsigned vreg[8], ks, vs[2][2 * GROUPS];
  bool dead = false;  // of the values on their way, no row sees some
  int dead_at = 0, dead_key = 0;
  bool dead_page = false;
  auto code_at = [&](int key, int page) {
    return (unsigned long long)(have(page) ? (unsigned)page : 0u) * c.page + (unsigned)((key & mask) * c.token);
  };
  auto word_at = [&](int key, int page) {
    return (unsigned long long)(have(page) ? (unsigned)page : 0u) * c.scale_page + (unsigned)((key & mask) * (2 * GROUPS));
  };
  auto fetch_k = [&](int s0, int page) {
    const int key = key_of((s0 >> 4) + wave);
    const auto rk = pool(kb + code_at(key, page)), rks = pool(ksb + word_at(key, page));
    if constexpr (KW == 4) {
      const v4i x = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rk, kcol, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) kreg[i] = x[i];
    } else {
      const int2 x = __builtin_bit_cast(int2, __builtin_amdgcn_raw_buffer_load_b64(rk, kcol, 0, 0));
      kreg[0] = x.x, kreg[1] = x.y;
    }
    if constexpr (GROUPS == 2) ks = __builtin_amdgcn_raw_buffer_load_b32(rks, krow * 4, 0, 0);
    else ks = __builtin_amdgcn_raw_buffer_load_b16(rks, krow * 2, 0, 0);
  };
  auto fetch_v = [&](int s0, int page) {
    const int block = (s0 >> 4) + wave, key = key_of(block);
    const auto rv = pool(vb + code_at(key, page)), rvs = pool(vsb + word_at(key, page));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (GROUPS == 2) {
        const v4i x = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rvs, h * 16, 32 * i, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) vs[i][j] = (unsigned)x[j];
      } else {
        const int2 x = __builtin_bit_cast(int2, __builtin_amdgcn_raw_buffer_load_b64(rvs, h * 8, 16 * i, 0));
        vs[i][0] = (unsigned)x.x, vs[i][1] = (unsigned)x.y;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (NDB == 4) vreg[i * 4 + j] = __builtin_amdgcn_raw_buffer_load_b16(rv, vcol, (8 * i + j) * c.token, 0);
        else vreg[i * 4 + j] = __builtin_amdgcn_raw_buffer_load_b8(rv, vcol, (8 * i + j) * c.token, 0);
      }
    }
    dead_at = block << 4, dead_key = key, dead_page = !have(page);
    dead = dead_page || dead_at + 16 > hi || (key < any_from && key + 16 > a.sinks);
  };
  // The numbers of keys, in KW / 2 parts, and of values: four parts for their pairs, NDB for the stores.
  auto swizzle = [](int r, int chunk) { return chunk ^ (r & 7); };
  const int kto = (wave * 16 + krow) * (DP * 2);
  S4Two ktwo;
  auto put_k = [&](int slot, int part) {
    if (part == 0) {
      ktwo.set(bits, 0, __builtin_amdgcn_perm(ks, ks, 0x01000100u));
      ktwo.set(bits, 1, __builtin_amdgcn_perm(ks, ks, GROUPS == 2 ? 0x03020302u : 0x01000100u));
    }
    v2h u[4], w[4];
    ktwo.values(bits, (unsigned)kreg[2 * part], u);
    ktwo.values(bits, (unsigned)kreg[2 * part + 1], w);
    const int chunk = (kbyte >> 3) + part;
    char* const to = lds + slot * BYTES + kto;
    *reinterpret_cast<v8h*>(to + swizzle(krow, chunk) * 16) = join8(u[0], u[2], w[0], w[2]);
    *reinterpret_cast<v8h*>(to + swizzle(krow, chunk + DP / 16) * 16) = join8(u[1], u[3], w[1], w[3]);
  };
  v2h vy[4][4];
  auto dead_v = [&] {  // what no row sees is not there: steps, which may be anything, become zeros
    if (__builtin_expect(dead, 0)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (i >> 2) * 8 + h * 4 + (i & 3), key = dead_key + at;
        if (dead_page || dead_at + at >= hi || (key < any_from && key >= a.sinks)) {
          if (GROUPS == 2) vs[i >> 2][i & 3] = 0;
          else vs[i >> 2][(i & 3) >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
        }
      }
    }
  };
  auto make_v = [&](int j) {
    const unsigned* const w = vs[j >> 1];
    S4Two two;
    if constexpr (GROUPS == 2) {
      const unsigned first = w[2 * (j & 1)], second = w[2 * (j & 1) + 1];
      two.set(bits, 0, __builtin_amdgcn_perm(second, first, 0x05040100u));
      two.set(bits, 1, __builtin_amdgcn_perm(second, first, 0x07060302u));
    } else {
      two.set(bits, 0, w[j & 1]);
      two.set(bits, 1, w[j & 1]);
    }
    two.values(bits, vreg[2 * j] | vreg[2 * j + 1] << 16, vy[j]);
  };
  auto put_v = [&](int slot, int i) {
    *reinterpret_cast<v8h*>(lds + 2 * BYTES + slot * BYTES + ((wave * NDB + i) * 64 + lane) * 16) = join8(vy[0][i], vy[1][i], vy[2][i], vy[3][i]);
  };

  float off = PA_EMPTY, den = 0.0f;
  v16f acc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;

  // 32 keys: the softmax of their scores into their probabilities, beside it the scores of the next 32 and the products of the 32
  // before, in bundles that the compiler keeps in order: a matrix instruction, then what runs beside it.  Their operands go
  // through a ring of RING registers of 16 bytes a lane, read from the LDS RING - 1 bundles ahead.  Scores are two bundles ahead of
  // the products at the end, so that their largest is there when the next 32 begin.
  constexpr int BUNDLES = 2 * KS, RING = 4;
  struct Half {
    v16f x;     // scores
    float top;  // the largest of them
    v8h pr[2];  // probabilities
  };
  v8h op[RING];
  const int klane = n * (DP * 2) + ((h ^ (n & 7)) << 4);
  auto is_score = [](int m) { return m <= BUNDLES - 4 ? (m & 1) == 0 : m == BUNDLES - 3; };
  auto number = [](int m) { return m <= BUNDLES - 4 ? m >> 1 : m == BUNDLES - 3 ? KS - 1 : m - KS; };
  // operand m of the 32 keys whose scores come from the keys at `k` and whose products are of the values at `v`
  auto read = [&](int m, int k, int v) {
    if (is_score(m)) op[m % RING] = *reinterpret_cast<const v8h*>(lds + ((k + klane) ^ (number(m) << 5)));
    else op[m % RING] = *reinterpret_cast<const v8h*>(lds + v + (number(m) * 64 + lane) * 16);
  };
  // `ahead`: whether the operands that the next 32 keys begin with may be read already, from k_next and v_next
  auto run = [&](Half& now, Half& next, v8h (&before)[2], int k, int v, bool ahead, int k_next, int v_next, auto beside) {
    if (__builtin_expect(__ballot(__builtin_fmaf(now.top, cl, off) > 15.0f) != 0, 0)) {
      // A new reference.  It moves by a whole number, so that what is relative to the old one is scaled without rounding.
      auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(now.top), __float_as_uint(now.top), false, false);
      const float top = __builtin_fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1]));
      const float above = __builtin_fmaf(top, cl, off) - 8.0f;
      const bool moves = above > 7.0f, first = off == PA_EMPTY;
      const float by = moves ? __builtin_ceilf(above) : 0.0f;
      const float scale = first && moves ? 0.0f : __builtin_amdgcn_exp2f(-by);
      off = !moves ? off : first ? __builtin_fmaf(-top, cl, 8.0f) : off - by;
      den *= scale;
      // (in two steps: a probability of 2^15 is still one of fp16 where it is to become 2^-20, the factor for it is not)
      const float part = __builtin_floorf(by * 0.5f);
      const _Float16 scale_1 = (_Float16)__builtin_amdgcn_exp2f(-part), scale_2 = (_Float16)__builtin_amdgcn_exp2f(part - by);
#pragma unroll
      for (int q = 0; q < 2; ++q) before[q] = before[q] * scale_1 * scale_2;
#pragma unroll
      for (int i = 0; i < NDB; ++i) acc[i] *= scale;
    }
    v16f t;
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] = 0.0f;
    float e[16];
    v2h two[8];
    constexpr int EACH = 16 / BUNDLES;  // scores to a bundle
    auto softmax = [&](int m) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int r = m * EACH + i;
        if (r < 16) e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(now.x[r], cl, off));
        if (r >= 3 && r < 19 && (r & 1)) {
          const v2f pair = {e[r - 3], e[r - 2]};
          two[(r - 3) >> 1] = __builtin_convertvector(pair, v2h);
          asm volatile("" : "+v"(two[(r - 3) >> 1]));  // computed here, not where the next 32 keys need it
        }
        if (r >= 4 && r < 20 && !(r & 1)) den = __builtin_amdgcn_fdot2(two[(r - 4) >> 1], v2h{(_Float16)1.0f, (_Float16)1.0f}, den, false);
      }
    };
#pragma unroll
    for (int m = 0; m < BUNDLES; ++m) {
      __builtin_amdgcn_sched_barrier(0);
      const int i = number(m);
      if (is_score(m)) t = __builtin_amdgcn_mfma_f32_32x32x16_f16(op[m % RING], qf[i], t, 0, 0, 0);
      else acc[i % NDB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(op[m % RING], before[i / NDB], acc[i % NDB], 0, 0, 0);
      softmax(m);
      if (m + RING - 1 < BUNDLES) read(m + RING - 1, k, v);
      else if (ahead) read(m + RING - 1 - BUNDLES, k_next, v_next);
      beside(m);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = BUNDLES; m * EACH < 20; ++m) softmax(m);
    next.top = t[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) next.top = __builtin_fmaxf(next.top, t[r]);
    asm volatile("" : "+v"(den), "+v"(next.top));
    next.x = t;
#pragma unroll
    for (int q = 0; q < 2; ++q) now.pr[q] = join8(two[4 * q], two[4 * q + 1], two[4 * q + 2], two[4 * q + 3]);
  };

  if (lo < hi) {
    // whether the pool lacks any of the item's pages: looked at once, so that steps need not
    bool holes = false;
    for (int i = (lo >> 4) + lane; i <= last_block; i += 64) holes |= !have(table[key_of(i) >> c.page_shift]);
    holes = __ballot(holes) != 0;
    // Pages are looked up a step ahead, by vector loads: these return in order, so that the wait for the keys and values in
    // front of one is all the wait it needs (a scalar one would have to be over at every wait for the LDS).
    int zero = 0;
    asm("" : "+v"(zero));
    auto ask = [&](int s0) { return b.table[(long long)it.seq * b.per_seq + (key_of((s0 >> 4) + wave) >> c.page_shift) + zero]; };
    auto page_at = [&](int s0) { return table[key_of((s0 >> 4) + wave) >> c.page_shift]; };
    const int page0 = page_at(lo), page1 = page_at(lo + ST_KEYS);
    int asked = ask(lo + 2 * ST_KEYS);
    fetch_k(lo, page0);
    fetch_v(lo, page0);
    if (c.D < DP) {  // chunks behind the head size are never written: zeros, as Q is there
      for (int i = threadIdx.x * 16; i < 2 * BYTES; i += PA_THREADS * 16) *reinterpret_cast<v4i*>(lds + i) = v4i{0, 0, 0, 0};
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < KW / 2; ++i) put_k(0, i);
    fetch_k(lo + ST_KEYS, page1);
    dead_v();
#pragma unroll
    for (int j = 0; j < 4; ++j) make_v(j);
#pragma unroll
    for (int i = 0; i < NDB; ++i) put_v(0, i);
    fetch_v(lo + ST_KEYS, page1);
    __syncthreads();
    // keys whose scores do not count: masks, and pages that are lost
    auto hide = [&](v16f& x, float& top, int s0) {
      const int k0 = key_of(s0 >> 4), k1 = key_of((s0 >> 4) + 1);
      if (__builtin_expect(s0 + 32 > hi || k1 + 15 > w0 || k0 < wave_all_from || holes, 0)) {
        bool on[2] = {true, true};
        if (holes) on[0] = have(table[k0 >> c.page_shift]), on[1] = have(table[k1 >> c.page_shift]);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = (r & 3) + 8 * ((r >> 2) & 1) + 4 * h, mine = (r >> 3 ? k1 : k0) + at;
          if (s0 + 16 * (r >> 3) + at >= hi || mine >= limit || !on[r >> 3] || (mine < from && mine >= a.sinks)) x[r] = -__builtin_inff();
        }
        top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = __builtin_fmaxf(top, x[r]);
      }
    };
    Half even, odd;
    {
      v16f t;
#pragma unroll
      for (int r = 0; r < 16; ++r) t[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
        t = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const v8h*>(lds + (klane ^ (i << 5))), qf[i], t, 0, 0, 0);
      even.x = t;
      even.top = t[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) even.top = __builtin_fmaxf(even.top, t[r]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) odd.pr[q][j] = (_Float16)0.0f;
    // A step is 64 keys, in two halves.  Beside the first: the scores of the second, the products of the second half before it (in the
    // first step of its own, times zero), and keys of the next step become numbers.  Beside the second: the scores of the next step's
    // first half, the products of the first, and values of the next step become numbers.  Keys and values have two places each; the
    // barrier between the halves makes sure that what the second reads is there, and that what is written behind it has been read.
    constexpr int K_HALF = 32 * DP * 2, V0 = 2 * BYTES, V_HALF = BYTES / 2;
    int slot = 0, v_before = V0 + V_HALF;
#pragma unroll
    for (int m = 0; m < RING - 1; ++m) read(m, K_HALF, v_before);
    int s0 = lo, page = 0;
    for (;;) {
      const int other = slot ^ 1, k_other = other * BYTES, v_now = V0 + slot * BYTES;
      // the same for all lanes: with the half behind its last keys a wave gathers those
      const bool here = __builtin_amdgcn_readfirstlane(s0 < keys + 32) != 0;
      auto stage_k = [&](int m) {
        if (m == 0) page = __builtin_amdgcn_readfirstlane(asked);
#pragma unroll
        for (int i = 0; i < KW / 2; ++i)
          if (m == KS / 2 + i * (KS / 4)) put_k(other, i);
        if (m == BUNDLES - 2) {
          fetch_k(s0 + 2 * ST_KEYS, page);
          asked = ask(s0 + 3 * ST_KEYS);
        }
      };
      auto stage_v = [&](int m) {
        if (m == KS / 4) dead_v();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (m == KS / 4 + j * (KS / 4)) make_v(j);
#pragma unroll
        for (int i = 0; i < NDB; ++i)
          if (m == KS + KS / 4 + (i * KS / 4) / (NDB / 2)) put_v(other, i);
        if (m == BUNDLES - 1) fetch_v(s0 + 2 * ST_KEYS, page);
      };
      if (__builtin_expect(here, 1)) {
        hide(even.x, even.top, s0);
        run(even, odd, odd.pr, slot * BYTES + K_HALF, v_before, false, 0, 0, stage_k);
      } else {
#pragma unroll
        for (int m = 0; m < BUNDLES; ++m) stage_k(m);
      }
      __syncthreads();
      if (__builtin_expect(here, 1)) {
#pragma unroll
        for (int m = 0; m < RING - 1; ++m) read(m, k_other, v_now);
        hide(odd.x, odd.top, s0 + 32);
        run(odd, even, even.pr, k_other, v_now, true, k_other + K_HALF, v_now + V_HALF, stage_v);
      } else {
#pragma unroll
        for (int m = 0; m < BUNDLES; ++m) stage_v(m);
      }
      v_before = v_now + V_HALF;
      slot = other;
      s0 += ST_KEYS;
      if (s0 >= hi) break;
    }
    if (s0 < keys + 32) {  // nobody has gathered them: the wave's keys reach into the last half
#pragma unroll
      for (int i = 0; i < KS; ++i)
        acc[i % NDB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const v8h*>(lds + v_before + (i * 64 + lane) * 16),
                                                              odd.pr[i / NDB], acc[i % NDB], 0, 0, 0);
    }
  }

  // the two halves of the wave add their denominators
  {
    auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(den), __float_as_uint(den), false, false);
    den = __uint_as_float(o[0]) + __uint_as_float(o[1]);
  }
  // Through the LDS, four places at a spot that the row moves, so that rows leave as whole lines.
  __syncthreads();
  const float f = it.splits > 1 ? 1.0f : den != 0.0f ? a.alpha_pv / den : 0.0f;
  constexpr int QUADS = DP / 4, PER = 64 / QUADS;  // rows that a wave stores at once
  v4f* const own = reinterpret_cast<v4f*>(lds) + wave * 32 * QUADS;
  auto spot = [](int r, int quad) { return r * QUADS + (quad ^ (r & (QUADS - 1))); };
#pragma unroll
  for (int nib = 0; nib < 2; ++nib)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[NDB / 2][4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < NDB / 2; ++j) {
          const int at = r * (NDB / 2) + j;
          y[at >> 2][at & 3] = den != 0.0f ? acc[2 * j + nib][4 * i + r] * f : 0.0f;
        }
#pragma unroll
      for (int j = 0; j < NDB / 2; ++j)
        own[spot(n, nib * (QUADS / 2) + (2 * i + h) * (NDB / 2) + j)] = v4f{y[j][0], y[j][1], y[j][2], y[j][3]};
    }
  __builtin_amdgcn_wave_barrier();
  const long long place = it.place + (long long)it.split * it.step;
  const int quad = lane % QUADS, column = paged_column<DP>(quad * 4, c.D);
  const PagedRows out_row(it, a.q_heads, G, ST_ROWS);
#pragma unroll
  for (int i = 0; i < 32 / PER; ++i) {
    const int r = i * PER + lane / QUADS, rr = row0 + r;
    if (rr >= live_rows || column >= c.D) continue;
    const v4f y = own[spot(r, quad)];
    if (it.splits == 1) store_some<4, OUT>(a.out, out_row(wave * 32 + r) * c.D + column, {y[0], y[1], y[2], y[3]});
    else *reinterpret_cast<v4f*>(p.ws + (place * ST_ROWS + wave * 32 + r) * DP + quad * 4) = y;
  }
  if (it.splits > 1 && real && h == 0)
    *reinterpret_cast<v2f*>(p.ws + (long long)p.places * ST_ROWS * DP + (place * ST_ROWS + wave * 32 + n) * 2) = v2f{off, den};
}

// (two groups of a wide head take 144 registers, three waves to a SIMD; four would spill)
template <int DP, int GROUPS, int OUT>
__global__ __launch_bounds__(PA_THREADS, DP == 128 && GROUPS == 2 ? 3 : 4) void paged_attn_s4_rows_kernel(PagedAttn4 a, PagedCache4 c,
                                                                                                         PagedBatch b, PagedPlan rows) {
  __shared__ __attribute__((aligned(16))) char lds[s4_rows_lds(DP)];
  const int lo = b.cu[0], hi = b.cu[b.seqs];  // (on their way beside what the item needs)
  s4_rows<DP, GROUPS, OUT>(a, c, b, rows, blockIdx.x, lds);
  if (a.fill) paged_fill(b, lo, hi, static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
}

// Sequences of few rows and of many in one launch, 256 items of the one kind after 256 of the other as long as both last (as over the
// int8 cache, where turns of 256 leave one of each kind to every CU).
constexpr int S4_TURN = 256;
template <int DP, int GROUPS, int OUT>
__global__ __launch_bounds__(PA_THREADS, 2) void paged_attn_s4_both_kernel(PagedAttn4 a, PagedCache4 c, PagedBatch b, PagedPlan rows,
                                                                           PagedPlan tiles) {
  __shared__ __attribute__((aligned(16))) char lds[s4_tiles_lds(DP) > s4_rows_lds(DP) ? s4_tiles_lds(DP) : s4_rows_lds(DP)];
  if (a.fill) paged_fill(b, b.cu[0], b.cu[b.seqs], static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
  const int i = blockIdx.x, each = (rows.slots < tiles.slots ? rows.slots : tiles.slots) & -S4_TURN, rest = i - 2 * each;
  bool many = rest < 0 ? (i & S4_TURN) == 0 : rest < tiles.slots - each;
  int index = rest < 0 ? i / (2 * S4_TURN) * S4_TURN + i % S4_TURN : each + rest - (many ? 0 : tiles.slots - each);
  if (b.seqs == 1) many = paged_seq(b, c.page_shift, 0).T * rows.group > PA_ROWS, index = i;  // of one kind
  if (many) s4_tiles<DP, GROUPS, OUT>(a, c, b, tiles, index, lds);
  else s4_rows<DP, GROUPS, OUT>(a, c, b, rows, index, lds);
}

// Joins slices that do not meet in the launch itself, EACH rows to a workgroup, in turns of eight items (as over the int8 cache): the
// many rows', which take longer, in the first `tile_blocks` workgroups, the few rows' in the others.
constexpr int S4_JOIN = 2;
template <int ROWS, int EACH, int DP, int OUT>
__device__ __forceinline__ void s4_join(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const PagedPlan& p, int block, float* meet) {
  constexpr int PIECES = ROWS / EACH;
  const int index = block / (8 * PIECES) * 8 + block % 8;
  PagedItem it;
  if constexpr (ROWS == ST_ROWS) it = paged_item<ST_PARTS, true, false, S4_HELD>(b, c.page_shift, c.heads, ROWS, p, index);
  else it = paged_item<4, true, true, S4_HELD>(b, c.page_shift, c.heads, ROWS, p, index);
  if (!it.found || it.split != 0) return;
  join_slices<ROWS, EACH, DP, OUT, false, true>(PagedOut{a.out, a.q_heads, c.D, a.alpha_pv}, p, it, meet, block / 8 % PIECES * EACH);
}
template <int DP, int OUT>
__global__ __launch_bounds__(PA_THREADS) void paged_attn_s4_join_kernel(PagedAttn4 a, PagedCache4 c, PagedBatch b, PagedPlan rows,
                                                                        PagedPlan tiles, int tile_blocks) {
  __shared__ __attribute__((aligned(16))) float meet[PA_THREADS * 8];
  const int block = blockIdx.x;
  if (block < tile_blocks) s4_join<ST_ROWS, ST_JOIN, DP, OUT>(a, c, b, tiles, block, meet);
  else s4_join<PA_ROWS, S4_JOIN, DP, OUT>(a, c, b, rows, block - tile_blocks, meet);
}

// Slices that the keys of a batch are cut into, about: three to a CU.  An item is cut where it has one and a half times as many keys or
// more, into even parts, and longer slices come first.  75 tokens over 50 to 7003 keys, 8 key heads of four, take 105 us with 512
// slices of one length each and a rest, none where 512 items fill the chip (the int8 cache's rule, whose kernel waits for memory
// longer), 83 without that exception, 75 with even ones, long ones first; 512, 768 and 1024 slices of them 80, 75 and 75, 20 x 4 tokens
// in windows of 1024 keys 29, 29 and 34 (where 768 leave 640 items whole).
constexpr int S4_TARGET = 768;

// Rows to a sequence, on average, up to which all of a batch go to the kernel of 16 rows: it reads a sequence's keys once for every 16,
// but starts sooner, spreads further and has three or four waves to a SIMD.  All by it, and by tiles: 16 sequences of 500 to 4000 keys, 32
// heads on 8, 8 tokens each (32 rows) 28 and 55 us, 12 (48) 32 and 58, 16 (64) 38 and 59.  A chunk among single tokens, which this sends to the
// same kernel, gains where it is short or its keys are few, and loses otherwise: all by this kernel, and by both, 32 heads on 8, 250 and 500
// tokens beside 60 over up to 3000 keys 73 and 105 us, and 87 and 97, 512 beside 63 over 2000, 6000 and 12000 80, 199 and 379, and 84, 168 and 288;
// own keys, 40 heads, 700 beside 31 over 2000, 6000 and 12000 119, 319 and 638, and 137, 293 and 519; 32 heads, 300 beside 15 over 4000 and 13000 91
// and 262, and 101 and 242, 700 beside 15 146 and 448, and 130 and 345.  A line that also knows the longest sequence would take the better of
// the two; the host knows no lengths.
constexpr int S4_FEW_MEAN = 48;

// Sequences of a batch of the other kind up to which those of few rows are cut into S4_TARGET slices as well; of more, into 128, since
// they share the chip with tiles.  So few can be all there is, the rest being rows of nobody behind a recorded step: one token over 200000
// keys and 3 such rows, 16 heads on 1, 32 us, 349 when one sequence went to the tiles; 4 tokens over 50000 and 30 rows, 64 on 8, 70 us, 123
// in 128 slices; 8 over 20000 and 50 rows 58 and 101.  Beside a chunk over 20000 keys, 32 heads on 8, it pays
// for 7 single tokens too (chunks of 100, 512 and 2000 tokens 129, 253 and 776 us; 185, 315 and 776), for 15 it depends (900 tokens 424 and
// 472, 2500 tokens 1012 and 991).
constexpr int S4_LONE = 8;

// What a call of these sizes runs: bounds, since the lengths are on the device (see the int8 cache's).
struct S4Kind {
  long long items;   // at most
  long long slots;   // the same, slices included; 0: none of this kind
  long long places;  // slices of those that are cut
  int target;        // slices that the keys are cut into; 0: nothing is cut
  void cut(int into, long long of_one) {
    target = into;
    // an item has at most as many slices as there are shortest ones in it, all together `target` more than items
    const long long most = items * (of_one - 1);
    slots += most < target + 8 ? most : target + 8;
    places = slots < 2 * target + 8 ? slots : 2 * target + 8;
  }
};
struct S4Shape {
  S4Kind rows, tiles;
  bool meet;  // slices of few rows meet in the launch
};
static S4Shape s4_shape(long long rows, long long seqs, long long group, long long heads, long long capacity) {
  S4Shape s = {};
  const bool cut = seqs > 0 && capacity >= PA_MIN_SLICE + PA_MIN_SLICE / 2;
  const long long of_one = capacity / PA_MIN_SLICE + 1;  // slices of one item
  long long each = PA_ROWS;                              // rows of one
  auto items = [](S4Kind& k, long long n) { k.items = k.slots = n; };
  auto join_here = [&] {
    const long long shared = s.rows.target / (s.rows.items > 0 ? s.rows.items : 1) + 1;
    s.meet = s.rows.target > 0 && (of_one < shared ? of_one : shared) * each * 520 <= 66560;
  };
  if (rows * group <= S4_FEW_MEAN * seqs) {  // few rows to a sequence on average, nobody's counted: all of them by that kernel
    items(s.rows, heads * (seqs + rows * group / PA_ROWS));
    each = rows * group / (seqs > 0 ? seqs : 1) + 1 < PA_ROWS ? rows * group / (seqs > 0 ? seqs : 1) + 1 : PA_ROWS;
    if (cut) s.rows.cut(S4_TARGET, of_one);
    join_here();
    return s;
  }
  // sequences with more than 16 rows are at most a 17th of all rows
  const long long many = rows * group / (PA_ROWS + 1) < seqs ? rows * group / (PA_ROWS + 1) : seqs;
  items(s.tiles, heads * (many + rows * group / ST_ROWS));
  if (cut && s.tiles.items < ST_PLENTY) s.tiles.cut(ST_TARGET, of_one);
  // Rows can be nobody's: one sequence too may have 16 of them or fewer.
  items(s.rows, heads * seqs);
  if (cut) s.rows.cut(seqs <= S4_LONE ? S4_TARGET : PA_TARGET / 4, of_one);
  join_here();
  return s;
}
static int s4_dp(long long D) { return D <= 64 ? 64 : 128; }
static long long s4_bytes(const S4Kind& k, int rows, long long D) { return k.places * rows * (s4_dp(D) + 2) * 4; }

long long paged_attn_s4_arrivals(long long rows, long long seqs, long long q_heads, long long heads, long long capacity) {
  const S4Shape s = s4_shape(rows, seqs, q_heads / heads, heads, capacity);
  return s.meet ? s.rows.places : 0;
}
long long paged_attn_s4_workspace_bytes(long long rows, long long seqs, long long q_heads, long long heads, long long D,
                                        long long capacity) {
  const S4Shape s = s4_shape(rows, seqs, q_heads / heads, heads, capacity);
  return s4_bytes(s.rows, PA_ROWS, D) + s4_bytes(s.tiles, ST_ROWS, D);
}

template <int DP, int GROUPS, int OUT>
static void launch_s4(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const S4Shape& s, const PagedPlan& rows,
                      const PagedPlan& tiles, hipStream_t stream) {
  const int slots = b.seqs != 1 ? rows.slots + tiles.slots : rows.slots < tiles.slots ? tiles.slots : rows.slots;
  const unsigned grid = (unsigned)(slots > 0 ? slots : 1);
  if (tiles.slots > 0)
    hipLaunchKernelGGL((paged_attn_s4_both_kernel<DP, GROUPS, OUT>), dim3(grid), dim3(PA_THREADS), 0, stream, a, c, b, rows, tiles);
  else
    hipLaunchKernelGGL((paged_attn_s4_rows_kernel<DP, GROUPS, OUT>), dim3(grid), dim3(PA_THREADS), 0, stream, a, c, b, rows);
  // an item that is cut has more than a target-th of all keys, so there are fewer than `target` of them
  auto items = [](const S4Kind& k) { return (unsigned)((k.items < k.target ? (int)k.items : k.target) + 7 & ~7); };
  const unsigned row_blocks = rows.target > 0 && rows.arrivals == nullptr ? items(s.rows) * (PA_ROWS / S4_JOIN) : 0;
  const unsigned tile_blocks = tiles.target > 0 ? items(s.tiles) * (ST_ROWS / ST_JOIN) : 0;
  if (row_blocks + tile_blocks > 0)
    hipLaunchKernelGGL((paged_attn_s4_join_kernel<DP, OUT>), dim3(row_blocks + tile_blocks), dim3(PA_THREADS), 0, stream, a, c, b, rows, tiles,
                       (int)tile_blocks);
}

int launch_paged_attn_s4(int out_type, const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream) {
  if (b.rows == 0 || a.q_heads == 0) return TI_OK;
  const int group = a.q_heads / c.heads;
  const long long capacity = (long long)b.per_seq << c.page_shift;
  S4Shape s = s4_shape(b.rows, b.seqs, group, c.heads, capacity);
  const long long rows_bytes = s4_bytes(s.rows, PA_ROWS, c.D);
  if (workspace == nullptr || workspace_bytes < rows_bytes + s4_bytes(s.tiles, ST_ROWS, c.D))
    s.rows.target = s.tiles.target = 0, s.meet = false;
  const long long items = b.seqs != 1 ? s.rows.slots + s.tiles.slots : s.rows.slots < s.tiles.slots ? s.tiles.slots : s.rows.slots;
  if (items > 0x7fffff) return fail(TI_ERR_INVALID_ARG, "paged_attn_s4: %lld work items", items);
  auto plan = [&](const S4Kind& k, int rows_of_item, int least, int most, char* ws) {
    PagedPlan p;
    p.group = group;
    p.least = least;
    p.most = most;
    p.target = k.target;
    p.full = 0x7fffffff;
    p.at_once = rows_of_item == ST_ROWS ? ST_AT_ONCE : 0;
    p.even = true;
    // with a window an item reads its own keys, the first ones, and what its tokens' windows are apart
    const long long span = a.window > 0 ? (long long)a.window + ((a.sinks + 15) & ~15) + 16 + (rows_of_item + group - 1) / group + 1 : 0x7fffffff;
    p.span = span < 0x7fffffff ? (int)span : 0x7fffffff;
    p.slots = (int)k.slots;
    p.places = (int)k.places;
    p.ws = reinterpret_cast<float*>(ws);
    p.arrivals = nullptr;
    return p;
  };
  char* const ws = static_cast<char*>(workspace);
  PagedPlan rows = plan(s.rows, PA_ROWS, 0, s.tiles.slots > 0 ? PA_ROWS : 0x7fffffff, ws);
  const PagedPlan tiles = plan(s.tiles, ST_ROWS, s.rows.slots > 0 ? PA_ROWS : 0, 0x7fffffff, ws + (s.rows.target ? rows_bytes : 0));
  const bool meet = a.arrivals != nullptr && a.arrivals_count >= paged_attn_s4_arrivals(b.rows, b.seqs, a.q_heads, c.heads, capacity);
  rows.arrivals = meet && s.meet ? a.arrivals : nullptr;
  auto run = [&](auto dp, auto groups) {
    constexpr int DP = decltype(dp)::value, GROUPS = decltype(groups)::value;
    if (out_type == PT_S8) launch_s4<DP, GROUPS, PT_S8>(a, c, b, s, rows, tiles, stream);
    else if (out_type == PT_F16) launch_s4<DP, GROUPS, PT_F16>(a, c, b, s, rows, tiles, stream);
    else launch_s4<DP, GROUPS, PT_BF16>(a, c, b, s, rows, tiles, stream);
  };
  using std::integral_constant;
  if (s4_dp(c.D) == 64) {
    if (c.groups == 1) run(integral_constant<int, 64>(), integral_constant<int, 1>());
    else run(integral_constant<int, 64>(), integral_constant<int, 2>());
  } else {
    if (c.groups == 1) run(integral_constant<int, 128>(), integral_constant<int, 1>());
    else run(integral_constant<int, 128>(), integral_constant<int, 2>());
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_attn_s4 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

}  // namespace ti
