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

typedef int v4i_8 __attribute__((ext_vector_type(4), aligned(8)));  // 16 bytes at a multiple of 8

// A nibble in the low bits of a 16-bit half, or in the next four, is a number of fp16 with one bit operation: 0x6400 + u is 1024 + u,
// 0x5400 + 16 u is 64 + u.  Less the same with z, times the step: exact.  `c` has two bytes in each half (of two columns, or of two
// keys); the four results are the low byte's nibbles, then the high byte's.
struct S4Two {
  v2h step[2], base[2];  // of low nibbles and of high ones: the step, and 1024 + z or 64 + z
  __device__ __forceinline__ void set(int nibble, unsigned word) {  // `word`: a word in each half
    const unsigned s = word & 0x7ff07ff0u, z = (word & 0x000f000fu) | 0x64006400u;
    step[nibble] = __builtin_bit_cast(v2h, s);
    base[nibble] = __builtin_bit_cast(v2h, z);
    if (nibble) base[nibble] -= v2h{(_Float16)960.0f, (_Float16)960.0f};
  }
  __device__ __forceinline__ void values(unsigned c, v2h (&y)[4]) const {
    const unsigned d = c >> 8;
    const unsigned w[4] = {(c & 0x000f000fu) | 0x64006400u, (c & 0x00f000f0u) | 0x54005400u, (d & 0x000f000fu) | 0x64006400u,
                           (d & 0x00f000f0u) | 0x54005400u};
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (__builtin_bit_cast(v2h, w[i]) - base[i & 1]) * step[i & 1];
  }
};

__device__ __forceinline__ v8h join8(v2h a, v2h b, v2h c, v2h d) {
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// One element of a query as fp16.
__device__ __forceinline__ _Float16 query_at(const void* q, int type, long long i) {
  if (type == PT_S8) return (_Float16)(float)static_cast<const int8_t*>(q)[i];
  if (type == PT_F16) return static_cast<const _Float16*>(q)[i];
  return (_Float16)__uint_as_float((unsigned)static_cast<const uint16_t*>(q)[i] << 16);
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

// Few rows: 16 to a workgroup, its four waves take 32 keys each in turn.
constexpr int s4_rows_lds(int DP) { return PA_WAVES * PA_ROWS * (DP + 4 + 2) * 4; }
template <int DP, int GROUPS, int OUT>
__device__ __forceinline__ void s4_rows(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const PagedPlan& p, int index,
                                        char* lds) {
  constexpr int NB = DP / 16;  // column blocks; lane n of 16 has NB / 2 bytes of a value row, from NB / 2 * n on
  constexpr int KW = DP / 32;  // dwords of a key row that a lane has
  const auto sum = reinterpret_cast<float(*)[PA_ROWS][DP + 4]>(lds);
  const auto offs = reinterpret_cast<float(*)[PA_ROWS]>(lds + PA_WAVES * PA_ROWS * (DP + 4) * 4);
  const auto den = offs + PA_WAVES;

  const PagedItem it = paged_item<1>(b, c.page_shift, c.heads, PA_ROWS, p, index);
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
  // Q in the order in which a dword's nibbles come apart: bytes 0, 2, 1, 3.
  const int kbyte = kg * KW * 4 <= half - KW * 4 ? kg * KW * 4 : half - KW * 4;
  v8h qf[KW];  // of low nibbles, then of high ones
  {
    const long long from_q = (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head;
#pragma unroll
    for (int i = 0; i < KW; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int in = (i % (KW / 2)) * 8 + (j & 4) + ((j & 1) << 1 | (j & 2) >> 1), byte = kbyte + in;
        const bool there = real && byte >= kg * KW * 4 && byte < half;
        qf[i][j] = there ? query_at(a.q, a.q_type, from_q + byte + (i < KW / 2 ? 0 : half)) : (_Float16)0.0f;
      }
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const uint8_t* kb = c.k + it.head * c.k_head;
  const uint8_t* vb = c.v + it.head * c.v_head;
  const char* ksb = reinterpret_cast<const char*>(c.k_scale) + it.head * c.ks_head;
  const char* vsb = reinterpret_cast<const char*>(c.v_scale) + it.head * c.vs_head;
  // The table through the constant address space: nothing writes to it while the kernel runs, and scalar loads are counted
  // apart from the keys and values in flight, which a vector load would have to wait for.
  const auto table = (const __attribute__((address_space(4))) int*)(b.table + (long long)it.seq * b.per_seq);
  const int mask = (1 << c.page_shift) - 1, last_block = hi > 0 ? (hi - 1) >> 4 : 0;
  const int head_blocks = span.head >> 4, shift_blocks = span.shift >> 4;

  float off = PA_EMPTY;
  v4f acc[NB], dsum = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = v4f{0, 0, 0, 0};
  v8h ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (_Float16)1.0f;

  struct Step {
    int k[2][KW];
    unsigned v[8], ks[2], vs[2][2 * GROUPS];
    bool on[2];
  };
  auto block_of = [&](int s0, int blk) {  // blocks behind the last key are masked, and read where there is memory
    int at = (s0 >> 4) + blk;
    at = at < last_block ? at : last_block;
    return at < head_blocks ? at : at + shift_blocks;
  };
  auto pages_of = [&](int (&pg)[2], int s0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) pg[blk] = table[(block_of(s0, blk) << 4) >> c.page_shift];
  };
  const unsigned kcol = (unsigned)(n * c.k_token) + (unsigned)kbyte;
  const int vbyte = (n * NB / 2) & ~3;
  const unsigned vcol = (unsigned)(kg * 4 * c.v_token) + (vbyte < half ? (unsigned)vbyte : 0u);
  auto fetch = [&](Step& st, int s0, const int (&pg)[2]) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      int page = pg[blk];
      st.on[blk] = page >= 0 && page < c.pages;
      page = st.on[blk] ? page : 0;
      const int o = (block_of(s0, blk) << 4) & mask;
      const uint8_t* kr = kb + (long long)page * c.k_page + (long long)o * c.k_token + kcol;
      if constexpr (KW == 4) {
        const v4i x = *reinterpret_cast<const v4i_8*>(kr);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.k[blk][i] = x[i];
      } else {
        const int2 x = *reinterpret_cast<const int2*>(kr);
        st.k[blk][0] = x.x, st.k[blk][1] = x.y;
      }
      const char* kw = ksb + (long long)page * c.ks_page + (long long)(o + n) * (2 * GROUPS);
      st.ks[blk] = GROUPS == 2 ? *reinterpret_cast<const unsigned*>(kw) : *reinterpret_cast<const uint16_t*>(kw) * 0x10001u;
      const uint8_t* vr = vb + (long long)page * c.v_page + (long long)o * c.v_token + vcol;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        st.v[blk * 4 + j] = *reinterpret_cast<const unsigned*>(vr);
        vr += c.v_token;
      }
      const char* vw = vsb + (long long)page * c.vs_page + (long long)(o + kg * 4) * (2 * GROUPS);
      if constexpr (GROUPS == 2) {
        const v4i x = *reinterpret_cast<const v4i*>(vw);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.vs[blk][i] = (unsigned)x[i];
      } else {
        const int2 x = *reinterpret_cast<const int2*>(vw);
        st.vs[blk][0] = (unsigned)x.x, st.vs[blk][1] = (unsigned)x.y;
      }
    }
  };
  const unsigned vpick = DP == 128 || (n & 1) == 0 ? 0x05040100u : 0x07060302u;  // the half of a dword of V that this lane has
  auto work = [&](Step& st, int s0) {
    float x[8];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      S4Two k;
      k.set(0, __builtin_amdgcn_perm(st.ks[blk], st.ks[blk], 0x01000100u));
      k.set(1, __builtin_amdgcn_perm(st.ks[blk], st.ks[blk], 0x03020302u));
      v4f s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KW / 2; ++i) {
        v2h u[4], w[4];
        k.values((unsigned)st.k[blk][2 * i], u);
        k.values((unsigned)st.k[blk][2 * i + 1], w);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(u[0], u[2], w[0], w[2]), qf[i], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(join8(u[1], u[3], w[1], w[3]), qf[KW / 2 + i], s, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[blk * 4 + r] = s[r];
    }
    const int key0 = block_of(s0, 0) << 4, key1 = block_of(s0, 1) << 4;
    if (s0 + 32 > hi || key1 + 16 > p0 + 1 || key0 < all_from || !st.on[0] || !st.on[1]) {
      // What no row sees is not there: its values' steps, which may be anything, become zeros.
      auto dead = [&](int i) {
        const int key = (i >> 2 ? key1 : key0) + kg * 4 + (i & 3);
        return s0 + (i >> 2) * 16 + kg * 4 + (i & 3) >= hi || !st.on[i >> 2] || (key < any_from && key >= a.sinks);
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = (i >> 2 ? key1 : key0) + kg * 4 + (i & 3);
        if (dead(i) || key >= limit || (key < from && key >= a.sinks)) x[i] = -__builtin_inff();
        if (GROUPS == 2) {
          if (dead(i)) st.vs[i >> 2][i & 3] = 0;
        } else if (dead(i)) {
          st.vs[i >> 2][(i & 3) >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
        }
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = x[i] > top ? x[i] : top;
    // a new reference only where a probability would pass 2^15: it starts at 2^8, fp16 ends at 2^16
    if (__ballot(__builtin_fmaf(top, cl, off) > 15.0f) != 0) {
      top = rows_max(top);
      if (__builtin_fmaf(top, cl, off) > 15.0f) {
        const float fresh = 8.0f - top * cl;
        const float scale = __builtin_amdgcn_exp2f(fresh - off);
        off = fresh;
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] *= scale;
        dsum *= scale;
      }
    }
    v8h hi_p, lo_p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], cl, off));
      hi_p[i] = (_Float16)e;
      lo_p[i] = (_Float16)(e - (float)hi_p[i]);
    }
    dsum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, hi_p, dsum, 0, 0, 0);
    dsum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, lo_p, dsum, 0, 0, 0);
    S4Two v[4];  // of the keys' pairs
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned* const w = st.vs[j >> 1];
      if constexpr (GROUPS == 2) {
        const unsigned first = w[2 * (j & 1)], second = w[2 * (j & 1) + 1];
        v[j].set(0, __builtin_amdgcn_perm(second, first, 0x05040100u));
        v[j].set(1, __builtin_amdgcn_perm(second, first, 0x07060302u));
      } else {
        v[j].set(0, w[j & 1]);
        v[j].set(1, w[j & 1]);
      }
    }
#pragma unroll
    for (int h = 0; h < NB / 4; ++h) {
      v2h y[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j].values(__builtin_amdgcn_perm(st.v[2 * j + 1], st.v[2 * j], h ? 0x07060302u : vpick), y[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v8h vf = join8(y[0][i], y[1][i], y[2][i], y[3][i]);
        acc[4 * h + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, hi_p, acc[4 * h + i], 0, 0, 0);
        acc[4 * h + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, lo_p, acc[4 * h + i], 0, 0, 0);
      }
    }
  };

  int s0 = lo + wave * 32;
  if (s0 < hi) {
    constexpr int STRIDE = PA_WAVES * 32;
    Step even, odd;
    int pg[2];
    pages_of(pg, s0);
    fetch(even, s0, pg);
    pages_of(pg, s0 + STRIDE);
    for (;;) {  // a step's loads are issued without a branch around them, so that the waits can count them
      fetch(odd, s0 + STRIDE, pg);
      pages_of(pg, s0 + 2 * STRIDE);
      work(even, s0);
      s0 += STRIDE;
      if (s0 >= hi) break;
      fetch(even, s0 + STRIDE, pg);
      pages_of(pg, s0 + 2 * STRIDE);
      work(odd, s0);
      s0 += STRIDE;
      if (s0 >= hi) break;
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
  if (kg == 0) {
    offs[wave][n] = off;
    den[wave][n] = dsum[0];
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

template <int DP, int GROUPS, int OUT>
__global__ __launch_bounds__(PA_THREADS, 2) void paged_attn_s4_rows_kernel(PagedAttn4 a, PagedCache4 c, PagedBatch b, PagedPlan rows) {
  __shared__ __attribute__((aligned(16))) char lds[s4_rows_lds(DP)];
  const int lo = b.cu[0], hi = b.cu[b.seqs];  // (on their way beside what the item needs)
  s4_rows<DP, GROUPS, OUT>(a, c, b, rows, blockIdx.x, lds);
  if (a.fill) paged_fill(b, lo, hi, static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
}

// Joins slices that do not meet in the launch itself, EACH rows to a workgroup, in turns of eight items (as over the int8 cache).
template <int ROWS, int EACH, int DP, int OUT>
__global__ __launch_bounds__(PA_THREADS) void paged_attn_s4_join_kernel(PagedAttn4 a, PagedCache4 c, PagedBatch b, PagedPlan p) {
  __shared__ __attribute__((aligned(16))) float meet[PA_THREADS * 8];
  constexpr int PIECES = ROWS / EACH;
  const PagedItem it = paged_item<1, true>(b, c.page_shift, c.heads, ROWS, p, blockIdx.x / (8 * PIECES) * 8 + blockIdx.x % 8);
  if (!it.found || it.split != 0) return;
  join_slices<ROWS, EACH, DP, OUT, false, true>(PagedOut{a.out, a.q_heads, c.D, a.alpha_pv}, p, it, meet, blockIdx.x / 8 % PIECES * EACH);
}

// What a call of these sizes runs: bounds, since the lengths are on the device (see the int8 cache's).
struct S4Shape {
  long long slots;   // items, slices included
  long long places;  // slices of those that are cut
  int target;        // slices that the keys are cut into; 0: nothing is cut
  bool meet;         // slices meet in the launch
};
static S4Shape s4_shape(long long rows, long long seqs, long long group, long long heads, long long capacity) {
  S4Shape s = {heads * (seqs + rows * group / PA_ROWS), 0, 0, false};
  if (seqs > 0 && capacity > PA_MIN_SLICE) {
    s.target = PA_TARGET;
    const long long each = rows * group / seqs + 1 < PA_ROWS ? rows * group / seqs + 1 : PA_ROWS;
    s.meet = s.target * each * 520 <= 66560 * s.slots;
    s.slots += s.target + 8;
    s.places = s.slots < 2 * s.target + 8 ? s.slots : 2 * s.target + 8;
  }
  return s;
}
static int s4_dp(long long D) { return D <= 64 ? 64 : 128; }

long long paged_attn_s4_arrivals(long long rows, long long seqs, long long q_heads, long long heads, long long capacity) {
  const S4Shape s = s4_shape(rows, seqs, q_heads / heads, heads, capacity);
  return s.meet ? s.places : 0;
}
long long paged_attn_s4_workspace_bytes(long long rows, long long seqs, long long q_heads, long long heads, long long D,
                                        long long capacity) {
  return s4_shape(rows, seqs, q_heads / heads, heads, capacity).places * PA_ROWS * (s4_dp(D) + 2) * 4;
}

template <int DP, int GROUPS, int OUT>
static void launch_s4(const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, const PagedPlan& rows, hipStream_t stream) {
  const unsigned grid = (unsigned)(rows.slots > 0 ? rows.slots : 1);
  hipLaunchKernelGGL((paged_attn_s4_rows_kernel<DP, GROUPS, OUT>), dim3(grid), dim3(PA_THREADS), 0, stream, a, c, b, rows);
  if (rows.target > 0 && rows.arrivals == nullptr) {
    const int most = rows.slots - rows.target - 8;
    const unsigned items = (unsigned)((most < rows.target ? most : rows.target) + 7 & ~7);
    hipLaunchKernelGGL((paged_attn_s4_join_kernel<PA_ROWS, 2, DP, OUT>), dim3(items * (PA_ROWS / 2)), dim3(PA_THREADS), 0, stream, a,
                       c, b, rows);
  }
}

int launch_paged_attn_s4(int out_type, const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream) {
  if (b.rows == 0 || a.q_heads == 0) return TI_OK;
  const int group = a.q_heads / c.heads;
  const long long capacity = (long long)b.per_seq << c.page_shift;
  S4Shape s = s4_shape(b.rows, b.seqs, group, c.heads, capacity);
  if (workspace == nullptr || workspace_bytes < paged_attn_s4_workspace_bytes(b.rows, b.seqs, a.q_heads, c.heads, c.D, capacity))
    s.target = 0, s.meet = false;
  if (s.slots > 0x7fffff) return fail(TI_ERR_INVALID_ARG, "paged_attn_s4: %lld work items", s.slots);
  PagedPlan rows;
  rows.group = group;
  rows.least = 0;
  rows.most = 0x7fffffff;
  rows.target = s.target;
  // with a window an item reads its own keys, the first ones, and what its tokens' windows are apart
  const long long span = a.window > 0 ? (long long)a.window + ((a.sinks + 15) & ~15) + 16 + (PA_ROWS + group - 1) / group + 1 : 0x7fffffff;
  rows.span = span < 0x7fffffff ? (int)span : 0x7fffffff;
  rows.slots = (int)s.slots;
  rows.places = (int)s.places;
  rows.ws = static_cast<float*>(workspace);
  const bool meet = a.arrivals != nullptr && a.arrivals_count >= paged_attn_s4_arrivals(b.rows, b.seqs, a.q_heads, c.heads, capacity);
  rows.arrivals = meet && s.meet ? a.arrivals : nullptr;
  auto run = [&](auto dp, auto groups) {
    constexpr int DP = decltype(dp)::value, GROUPS = decltype(groups)::value;
    if (out_type == PT_S8) launch_s4<DP, GROUPS, PT_S8>(a, c, b, rows, stream);
    else if (out_type == PT_F16) launch_s4<DP, GROUPS, PT_F16>(a, c, b, rows, stream);
    else launch_s4<DP, GROUPS, PT_BF16>(a, c, b, rows, stream);
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
