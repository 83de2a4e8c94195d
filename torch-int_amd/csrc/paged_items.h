// What the attentions over a paged KV cache share: work items that workgroups find for themselves, slices of long sequences and how
// they are joined, stores of contexts.
#pragma once
#include "paged.h"

namespace ti {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int PA_WAVES = 4;
constexpr int PA_ROWS = 16;
constexpr int PA_TARGET = 512;     // slices that the keys of a batch are cut into, beyond one to each item
constexpr int PA_FULL = 512;       // items that fill the chip
constexpr int PA_MIN_SLICE = 512;  // keys of a slice, at least
// Items are put in order where there are fewer than PA_SORTED of PA_LONG keys or more on average: finding one's own in four classes
// takes 1 to 4 us, which long items win back where few of them would end last.  Over the 4-bit cache, in order and as they come: 75 tokens
// over 50 to 7003 keys, 8 key heads, 75 and 82 us; 120 over 50 to 5000, 16 heads, 147 and 150; 64 over 3000 to 4000, 4 heads, 37.7 and 38.3; but
// 250 over 500 to 3000, 2 heads, 43 and 39; 200 over 20 to 3000, 8 heads, 88 and 86; 120 over 50 to 900, 8 heads, 28 and 26; 300 (which are
// looked at again for every class) over 20 to 1000, 8 heads, 98 and 62.
constexpr float PA_SORTED = 2048, PA_LONG = 2048;
constexpr float PA_EMPTY = 3.0e38f;  // offset of a row that has seen no key: 2^(-inf + PA_EMPTY) is 0

// The sequences that one of the two kernels takes, by how many rows a key head has in them, and how their keys are cut.
struct PagedPlan {
  int group;        // query heads of a key head
  int least, most;  // rows of a sequence: more than `least`, up to `most`
  int target;       // slices that the keys are cut into; 0: nothing is cut
  int full;         // items that fill the chip
  int at_once;      // workgroups that run at once, where slices are chosen for them to come out even; else 0
  bool even;        // slices of an item are of one length, up to half as long again, instead of the last one being what is left
  int span;         // keys that an item reads, at most
  int slots;        // work items at most, slices included: what the grid holds
  int places;       // slices of items that are cut, at most: what the workspace holds
  float* ws;        // partial sums [places][rows of an item][DP] fp32, then (offset, denominator) [places][rows]
  int* arrivals;    // [places] zeros, or null: a second launch joins the slices
  __device__ __forceinline__ int tiles(const PagedSeq& s, int rows_per_tile) const {
    const int rows = s.T * group;
    return rows > least && rows <= most ? (rows + rows_per_tile - 1) / rows_per_tile : 0;
  }
};

// Where contexts go: the output [rows, q_heads, D], packed, and the factor of the quotient of the sums.
struct PagedOut {
  void* out;
  int q_heads, D;
  float scale;
};

struct PagedItem {
  PagedSeq s;
  int seq, head, tile, split, splits;
  int place;  // of the slice 0 of an item that is cut, among all such slices (its others are `step` apart)
  int step;   // from one slice to the next: kv_heads * tiles
  int slice;  // keys of a slice
  bool found;
};

// Running sum over the lanes of a wave, in six steps through DPP: within rows of 16, then from row to row.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}
// The sum of all lanes, in every lane.
__device__ __forceinline__ float wave_add(float x) {
  auto step = [&](auto ctrl, auto rows) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
  step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The largest of the four lanes n, n + 16, n + 32, n + 48, in all of them.
__device__ __forceinline__ float rows_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Keys of a slice, the same in every workgroup: what cuts all keys of the batch into `target` equal parts.  Where the items
// alone fill the chip, only sequences of more than twice the average are cut: a slice costs its partial sums and the join.
__device__ __forceinline__ int paged_slice(float items, float total, int target, int full) {
  float want = total / (float)target;
  if (items >= (float)full) want = __builtin_fmaxf(want, 2.0f * total / items);
  const int slice = want < 1.0e9f ? ((int)want + 64) & ~63 : 1 << 30;
  return slice < PA_MIN_SLICE ? PA_MIN_SLICE : slice;
}

// The same for items of about one length that take long, `at_once` of them at a time: cut into as many slices as make the last round
// of workgroups least in vain.  A workgroup costs some 170 keys before and behind its own, one that is joined some 700.  Over the 4-bit cache, so and cut
// into `target` parts as above: 1536 rows over 6000 keys, 32 heads, 212 and 226 us; 700 over 13000, 28 heads on 4, 195 and 210; 300 rows and 31
// tokens over 600 to 2007, 32 heads on 8, 49.5 and 58; but 64 rows over 8000 53.7 and 51.8, 4 x 1000 rows over 4000 to 16000 931 and 847: of
// unequal items the longest ends last (and of more than 64 x HELD sequences nobody looks whether they are).  Those are cut into `target`
// parts, but none of fewer keys than make one round of all, nor of 2048: slices of at least 1024, 2048 and 4096 keys take 3 x 400 rows over
// 1500 to 5000 keys 123, 115 and 164 us, 2 x 200 over 5000 to 30000 223, 215 and 212; 16 x 24 rows over 500 to 4000 take 105 with 2048, 62
// with a round's; 16 x 100 over 400 to 900 83 without any, 61 so.
// Of items that are alike too, more than 16 slices have 2048 keys or more, as a join reads them one after another: 4 tokens over 200000 keys, 16
// heads on 1, 198 us, 289 with 1024, 375 with 16 slices at most; 32 tokens, 32 heads on 8, 237, 237 and 430; 8 x 40000, 16 on 1, 101, 98 and 112.
__device__ __forceinline__ int paged_slice_even(float items, float total, int target, int at_once) {
  const float keys = total / __builtin_fmaxf(items, 1.0f);
  float best = __builtin_ceilf(items / (float)at_once) * (keys + 170.0f);
  float slice = 2.0f * keys;
  // as many as there can be: of 512 keys up to 16, of PA_LONG beyond
  float most = __builtin_fmaxf(__builtin_fminf(keys / (float)PA_MIN_SLICE, 16.0f), keys / PA_LONG);
  most = __builtin_fminf(most, (float)target / __builtin_fmaxf(items, 1.0f));
  for (int rounds = 1; (rounds - 1) * at_once < target; ++rounds) {  // of all numbers that take as many rounds the largest costs least
    const float k = __builtin_floorf(__builtin_fminf((float)(rounds * at_once) / items, most));
    const float cost = __builtin_ceilf(items * k / (float)at_once) * (keys / k + 700.0f);
    if (k >= 2.0f && cost < best) best = cost, slice = keys / k;
  }
  const int want = slice < 1.0e9f ? ((int)slice + 63) & ~63 : 1 << 30;
  return want < PA_MIN_SLICE ? PA_MIN_SLICE : want;
}

// The work item with number `index`, in the order part, sequence, slice, tile of rows, head.  A sequence's tiles come from the
// last, which has the most keys, to the first, in PARTS parts, so that the long items of all sequences begin before the short
// ones.  SORTED: instead, in PARTS classes of sequences, those of long slices first.  CUT: the first slice of the `index`-th item
// among those that are cut.  HELD: 64 times so many sequences stay in registers, asked for together; of more, or with 1, 64 are
// looked at again at a time (over the 4-bit cache, 120 tokens over 50 to 900 keys, 8 key heads: 30 us, and 28 with 4).
template <int PARTS, bool CUT = false, bool SORTED = false, int HELD = 1>
__device__ __forceinline__ PagedItem paged_item(const PagedBatch& b, int page_shift, int heads, int rows_per_tile, const PagedPlan& p,
                                                int index) {
  PagedItem it;
  it.found = false;
  it.place = 0;
  if (b.seqs == 0) return it;
  const int lane = threadIdx.x & 63;
  PagedSeq s;
  int tiles;
  auto look = [&](int i0) {  // at sequence i0 + lane; behind the last one there is none
    s = PagedSeq{0, 0, 0, 0};
    tiles = 0;
    if (i0 + lane < b.seqs) {
      s = paged_seq(b, page_shift, i0 + lane);
      tiles = p.tiles(s, rows_per_tile);
    }
  };
  PagedSeq held[HELD];
  int held_tiles[HELD];
  const bool all = HELD > 1 && b.seqs <= 64 * HELD;
  if (all) {
    int lo[HELD], hi[HELD], len[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int i = h * 64 + lane < b.seqs ? h * 64 + lane : b.seqs - 1;
      lo[h] = b.cu[i], hi[h] = b.cu[i + 1], len[h] = b.lens[i];
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      held[h] = paged_seq(b, page_shift, lo[h], hi[h], len[h]);
      held_tiles[h] = h * 64 + lane < b.seqs ? p.tiles(held[h], rows_per_tile) : 0;
    }
    s = held[0], tiles = held_tiles[0];
  }
  it.slice = 0x7fffffff;
  bool sorted = false;
  if (p.target != 0) {
    auto keys_of = [&](const PagedSeq& s) { return (float)(s.len < p.span ? s.len : p.span); };
    float items = 0.0f, total = 0.0f;
    if (all) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) items += (float)held_tiles[h], total += (float)held_tiles[h] * keys_of(held[h]);
      items = wave_add(items), total = wave_add(total);
    } else {
      for (int i0 = (b.seqs - 1) & ~63; i0 >= 0; i0 -= 64) {  // the first 64 come last and stay
        look(i0);
        items += wave_add((float)tiles);
        total += wave_add((float)tiles * keys_of(s));
      }
    }
    bool alike = p.at_once != 0 && all;  // no item is longer than the average by more than a quarter
    if (alike)
#pragma unroll
      for (int h = 0; h < HELD; ++h) alike = alike && __ballot(held_tiles[h] > 0 && keys_of(held[h]) * items > 1.25f * total) == 0;
    const float count = items * (float)heads, keys = total * (float)heads;
    it.slice = alike ? paged_slice_even(count, keys, p.target, p.at_once) : paged_slice(count, keys, p.target, p.full);
    if (p.at_once != 0 && !alike) {  // (a joined slice costs 700)
      const float round = 1.25f * keys / (float)p.at_once;
      const int least = round < 4.0f * PA_MIN_SLICE ? (int)round & ~63 : 4 * PA_MIN_SLICE;
      it.slice = it.slice < least ? least : it.slice;
    }
    sorted = SORTED && count < PA_SORTED && total >= PA_LONG * items;
  }
  int before = 0, before_cut = 0, before_sliced = 0;
  int splits = 1;
  unsigned long long cuts = 0;  // which of the 64 sequences looked at are cut
  auto cut_up = [&] {
    const int keys = s.len < p.span ? s.len : p.span;
    const int over = p.even ? it.slice >> 1 : it.slice - 1;
    splits = keys <= it.slice ? 1 : (keys + over) / it.slice;
    cuts = __ballot(splits > 1 && tiles > 0);
  };
  if (b.seqs <= 64) {
    if (p.target == 0 && !all) look(0);
    cut_up();
    if (CUT && cuts == 0) return it;
  }
  const int parts = SORTED && !sorted ? 1 : PARTS;
  for (int part = 0, i0 = 0; part < parts; i0 + 64 < b.seqs ? i0 += 64 : (i0 = 0, ++part)) {
    if (b.seqs > 64) {
      if (all) {
#pragma unroll
        for (int h = 0; h < HELD; ++h)
          if (i0 == h * 64) s = held[h], tiles = held_tiles[h];
      } else {
        look(i0);
      }
      cut_up();
    }
    const int behind = PARTS == 1 || SORTED ? 0 : (int)((long long)tiles * part / PARTS);  // tiles of the parts before
    int here = PARTS == 1 || SORTED ? tiles : (int)((long long)tiles * (part + 1) / PARTS) - behind;
    if (sorted) {  // (four classes)
      const int keys = (s.len < p.span ? s.len : p.span) / splits, want = it.slice;
      const int mine = keys > want ? 0 : keys > (want >> 1) + (want >> 2) ? 1 : keys > want >> 1 ? 2 : 3;
      here = mine == part ? tiles : 0;
    }
    // a cu_new that descends can count rows many times over: no sum of items passes the range of int
    const long long whole = (long long)here * heads, slices = whole * splits;
    const int n = slices > 0x800000 ? 0x800000 : (int)slices;
    const int cut = splits == 1 ? 0 : whole > 0x800000 ? 0x800000 : (int)whole;
    const int upto = wave_scan(n), upto_cut = CUT ? wave_scan(cut) : 0;
    // what those of some lanes that are cut have of n, whose sum `all` is; mostly all of them are, or none
    auto sliced = [&](unsigned long long lanes, int all) {
      if ((cuts & lanes) == 0) return 0;
      if ((__ballot(n > 0) & lanes & ~cuts) == 0) return all;
      return __builtin_amdgcn_readlane(wave_scan((cuts & lanes) >> lane & 1 ? n : 0), 63);
    };
    const unsigned long long past = __ballot(CUT ? before_cut + upto_cut > index : before + upto > index);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int first = before + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at);
      const int rel = CUT ? index - (before_cut + __builtin_amdgcn_readlane(upto_cut, at) - __builtin_amdgcn_readlane(cut, at)) : index - first;
      const int t = __builtin_amdgcn_readlane(here, at), skip = __builtin_amdgcn_readlane(behind, at);
      it.s.row0 = __builtin_amdgcn_readlane(s.row0, at);
      it.s.T = __builtin_amdgcn_readlane(s.T, at);
      it.s.len = __builtin_amdgcn_readlane(s.len, at);
      it.splits = __builtin_amdgcn_readlane(splits, at);
      if (p.even) {
        const int keys = it.s.len < p.span ? it.s.len : p.span;
        it.slice = it.splits > 1 ? ((keys + it.splits - 1) / it.splits + 63) & ~63 : 0x7fffffff;
      }
      it.seq = i0 + at;
      it.step = heads * t;
      it.split = rel / it.step;
      const int rest = rel - it.split * it.step, from_last = rest / heads;
      it.tile = __builtin_amdgcn_readlane(tiles, at) - 1 - skip - from_last;
      it.head = rest - from_last * heads;
      it.found = it.split < it.splits && it.tile >= 0;
      if (it.splits > 1) {
        it.place = before_sliced + sliced((1ull << at) - 1, first - before) + rest;
        // all slices have a workgroup and a place, or (as a cu_new that descends can have it) the item is left out
        const long long behind_first = (long long)(it.splits - 1) * it.step;
        it.found = it.found && first + rest + behind_first < p.slots && it.place + behind_first < p.places;
      }
      return it;
    }
    const int sum = __builtin_amdgcn_readlane(upto, 63);
    before_sliced += sliced(~0ull, sum);
    before_sliced = before_sliced > 0x20000000 ? 0x20000000 : before_sliced;
    before += sum;
    before = before > 0x20000000 ? 0x20000000 : before;
    if (CUT) {
      before_cut += __builtin_amdgcn_readlane(upto_cut, 63);
      before_cut = before_cut > 0x20000000 ? 0x20000000 : before_cut;
    }
  }
  return it;
}

// Rows of no sequence (behind the last one; in front of the first, should it not begin at row 0) become zeros.  lo, hi: the first
// and the last entry of cu.
__device__ __forceinline__ void paged_fill(const PagedBatch& b, int lo, int hi, char* out, long long row_bytes) {
  lo = lo < 0 ? 0 : lo > b.rows ? b.rows : lo;
  hi = hi < lo ? lo : hi > b.rows ? b.rows : hi;
  const int rest = b.rows - (hi - lo);
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    char* at = out + (long long)(i < lo ? i : hi + i - lo) * row_bytes;
    for (long long j = threadIdx.x * 16ll; j < row_bytes; j += blockDim.x * 16ll) *reinterpret_cast<v4i*>(at + j) = v4i{0, 0, 0, 0};
  }
}

// Where the rows of a tile are in the output: row r of it is token (r0 + r) / group, head (r0 + r) % group.  The quotient comes
// from a multiplication: r0 + r < 4096 + 128 is small enough for it to be exact.
struct PagedRows {
  long long out0;   // output row of the tile's first token and of the key head's first query head
  int group, rest, step;
  float inv;
  __device__ __forceinline__ PagedRows(const PagedItem& it, int q_heads, int G, int rows_per_tile) : group(G), step(q_heads) {
    const int first = it.tile * rows_per_tile, t0 = first / G;
    rest = first - t0 * G;
    out0 = (long long)(it.s.row0 + t0) * q_heads + it.head * G;
    inv = 1.0f / (float)G;
  }
  __device__ __forceinline__ long long operator()(int r) const {
    const int x = rest + r, t = (int)(((float)x + 0.5f) * inv);
    return out0 + (long long)t * step + (x - t * group);
  }
};

// N neighbouring outputs (2 or 4)
template <int N, int OUT>
__device__ __forceinline__ void store_some(void* out, long long at, const float (&y)[N]) {
  if constexpr (OUT == PT_S8) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) w |= (unsigned)(rne_s8(y[i]) & 255) << (8 * i);
    if constexpr (N == 4) reinterpret_cast<unsigned*>(static_cast<int8_t*>(out) + at)[0] = w;
    else reinterpret_cast<unsigned short*>(static_cast<int8_t*>(out) + at)[0] = (unsigned short)w;
  } else {
    unsigned short h[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (OUT == PT_F16) {
        const _Float16 v = (_Float16)y[i];
        __builtin_memcpy(&h[i], &v, 2);
      } else {
        const __bf16 v = (__bf16)y[i];
        __builtin_memcpy(&h[i], &v, 2);
      }
    }
    unsigned w[N / 2];
    __builtin_memcpy(w, h, 2 * N);
    unsigned* to = reinterpret_cast<unsigned*>(static_cast<unsigned short*>(out) + at);
    if constexpr (N == 4) *reinterpret_cast<v2u*>(to) = v2u{w[0], w[1]};
    else to[0] = w[0];
  }
}

// Partial sums are written and read past the cache of the XCD: another XCD's workgroup may join them.
__device__ __forceinline__ void put4(float* p, float x, float y, float z, float w) {
  const v4f v = {x, y, z, w};
  asm volatile("global_store_dwordx4 %0, %1, off sc1" ::"v"(p), "v"(v) : "memory");
}
__device__ __forceinline__ void put2(float* p, float x, float y) {
  const unsigned long long w = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <bool THROUGH>
__device__ __forceinline__ float2 get2(const float* p) {
  if constexpr (!THROUGH) return *reinterpret_cast<const float2*>(p);
  const unsigned long long w =
      __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((unsigned)w), __uint_as_float((unsigned)(w >> 32)));
}

// A row's partial sums y relative to the offset `off`, with their denominator, and how two of them add up.
struct PagedPart {
  float off, den;
  v4f y;
  __device__ __forceinline__ void add(float o, float d, const v4f& x) {
    const float least = o < off ? o : off;
    const float mine = __builtin_amdgcn_exp2f(least - off), theirs = __builtin_amdgcn_exp2f(least - o);
    off = least;
    den = den * mine + d * theirs;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = y[i] * mine + x[i] * theirs;
  }
};

// Column of a place in a row of two halves of DP / 2 places, or D where there is none.
template <int DP>
__device__ __forceinline__ int paged_column(int d, int D) {
  const int at = d < DP / 2 ? d : d - DP / 2;
  return at >= D / 2 ? D : d < DP / 2 ? at : at + D / 2;
}

constexpr int PA_THREADS = PA_WAVES * 64;
// The slices of one item, COUNT of its ROWS rows from `first` on, by the threads of one workgroup.  A place is four
// columns of a row.  Its slices add up in four chains, every fourth slice to one, by four threads that meet in the LDS where
// places are few: the order, and the bits, are the same whoever joins.  HALVES: the places of a row are two halves of DP / 2, each
// with half of its columns.
constexpr int CHAINS = 4;
template <int ROWS, int COUNT, int DP, int OUT, bool THROUGH, bool HALVES = false>
__device__ __forceinline__ void join_slices(const PagedOut& to, const PagedPlan& p, const PagedItem& it, float* meet, int first) {
  const int G = p.group, tid = threadIdx.x;
  const int live_rows = it.s.T * G - it.tile * ROWS - first;
  const int rows = COUNT < live_rows ? COUNT : live_rows;
  if (rows <= 0) return;
  constexpr int QUADS = DP / 4;  // places of a row; those beyond the head size are idle
  const int work = rows * QUADS;
  const float* tail = p.ws + (long long)p.places * ROWS * DP;
  const PagedRows out_row(it, to.q_heads, G, ROWS);
  const PagedPart none = {PA_EMPTY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
  auto take = [&](PagedPart& sum, int e, int s) {
    const long long row = (it.place + (long long)s * it.step) * ROWS + first + e / QUADS;
    const float* from = p.ws + row * DP + e % QUADS * 4;
    const float2 od = get2<THROUGH>(tail + row * 2);
    if constexpr (THROUGH) {
      const float2 y0 = get2<true>(from), y1 = get2<true>(from + 2);
      sum.add(od.x, od.y, v4f{y0.x, y0.y, y1.x, y1.y});
    } else {
      sum.add(od.x, od.y, *reinterpret_cast<const v4f*>(from));
    }
  };
  auto give = [&](const PagedPart& sum, int e) {
    const int r = first + e / QUADS;
    int d = e % QUADS * 4;
    if constexpr (HALVES) d = paged_column<DP>(d, to.D);
    if (d >= to.D) return;
    const float f = sum.den != 0.0f ? to.scale / sum.den : 0.0f;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = sum.den != 0.0f ? sum.y[i] * f : 0.0f;
    store_some<4, OUT>(to.out, out_row(r) * to.D + d, y);
  };
  if (work * CHAINS <= PA_THREADS) {
    const int share = tid / work, e = tid - share * work;
    PagedPart sum = none;
    if (share < CHAINS) {
#pragma unroll 4
      for (int s = share; s < it.splits; s += CHAINS) take(sum, e, s);
    }
    float* mine = meet + tid * 8;
    mine[0] = sum.off, mine[1] = sum.den;
    *reinterpret_cast<v4f*>(mine + 4) = sum.y;
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int o = 1; o < CHAINS; ++o) {
      const float* at = meet + (tid + o * work) * 8;
      sum.add(at[0], at[1], *reinterpret_cast<const v4f*>(at + 4));
    }
    give(sum, e);
    return;
  }
  for (int e = tid; e < work; e += PA_THREADS) {
    PagedPart sum[CHAINS] = {none, none, none, none};
    for (int s = 0; s < it.splits; s += CHAINS)
#pragma unroll
      for (int o = 0; o < CHAINS; ++o)
        if (s + o < it.splits) take(sum[o], e, s + o);
#pragma unroll
    for (int o = 1; o < CHAINS; ++o) sum[0].add(sum[o].off, sum[o].den, sum[o].y);
    give(sum[0], e);
  }
}

// The workgroup that arrives last joins the slices, in their order: the bits do not depend on who that is.  Partial sums are
// written through to memory and read from there, and the counter is a device-scope atomic, so no cache has to be written back
// or emptied (which would take the other workgroups' keys with it): a thread's stores have arrived when its count of them is zero.
// `scratch`: LDS of the workgroup that nobody reads any more.
template <int ROWS, int DP, int OUT, bool HALVES = false>
__device__ __forceinline__ void meet_and_join(const PagedOut& o, const PagedPlan& p, const PagedItem& it, int* seen, float* scratch) {
  if (p.arrivals == nullptr) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    seen[0] = __hip_atomic_fetch_add(p.arrivals + it.place, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (seen[0] == it.splits - 1) __hip_atomic_store(p.arrivals + it.place, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (seen[0] != it.splits - 1) return;
  join_slices<ROWS, ROWS, DP, OUT, true, HALVES>(o, p, it, scratch, 0);
}

}  // namespace ti
