// Causal attention of a batch's new tokens over a paged int8 cache.  With x = q . k_j (exact int32), c = alpha_qk log2(e):
//   ctx = alpha_pv * sum_j 2^(c x_j - M) v_j / sum_j 2^(c x_j - M)     over the positions j up to the token's own.
// One pass over the keys with a running reference M; the products with V are fp16 MFMA with fp32 sums: int8 values times 2^-10
// are exact in fp16, and a probability goes in as the sum of two fp16 numbers (22 bits), since this kernel waits for
// memory and not for the matrix pipe.  The denominator is summed by the same instruction from the same rounded numbers.
//
// The heads that share a key head are rows of one product: a row is (token t, head g of the group), r = t * group + g.
// A work item is (sequence, key head, 16 rows, a slice of the keys); its waves take 32 keys in turn, each with its own M,
// and meet in the LDS at the end.  K and V go from memory to registers in the shape the MFMA wants: for Kt-major scores
// S^T = K Q^T a lane's operand is 16 bytes of one key row, and since the order of the inner dimension is free a lane takes 32
// neighbouring bytes; S^T leaves a lane with the scores of keys 4 kg .. 4 kg + 3 of two blocks of 16 for its row, which is
// already the operand of O^T = V^T P^T; and V^T's operand, eight keys of a column, is gathered from eight rows of 8 bytes (lane n
// of 16 owns the columns 8 n .. 8 n + 7) with one v_perm per two values, which also widens bytes to 16 bits.
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
constexpr float PA_EMPTY = 3.0e38f;  // offset of a row that has seen no key: 2^(-inf + PA_EMPTY) is 0

// The sequences that one of the two kernels takes, by how many rows a key head has in them, and how their keys are cut.
struct PagedPlan {
  int group;        // query heads of a key head
  int least, most;  // rows of a sequence: more than `least`, up to `most`
  int target;       // slices that the keys are cut into; 0: nothing is cut
  int slots;        // work items at most, slices included: what the grid holds
  int places;       // slices of items that are cut, at most: what the workspace holds
  float* ws;        // partial sums [places][rows of an item][DP] fp32, then (offset, denominator) [places][rows]
  int* arrivals;    // [places] zeros, or null: a second launch joins the slices
  __device__ __forceinline__ int tiles(const PagedSeq& s, int rows_per_tile) const {
    const int rows = s.T * group;
    return rows > least && rows <= most ? (rows + rows_per_tile - 1) / rows_per_tile : 0;
  }
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
__device__ __forceinline__ int paged_slice(float items, float total, int target) {
  float want = total / (float)target;
  if (items >= (float)PA_FULL) want = __builtin_fmaxf(want, 2.0f * total / items);
  const int slice = want < 1.0e9f ? ((int)want + 64) & ~63 : 1 << 30;
  return slice < PA_MIN_SLICE ? PA_MIN_SLICE : slice;
}

// The work item with number `index`, in the order part, sequence, slice, tile of rows, head.  A sequence's tiles come from the
// last, which has the most keys, to the first, in PARTS parts, so that the long items of all sequences begin before the short
// ones.  CUT: the first slice of the `index`-th item among those that are cut.
template <int PARTS, bool CUT = false>
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
  it.slice = 0x7fffffff;
  if (p.target != 0) {
    float items = 0.0f, total = 0.0f;
    for (int i0 = (b.seqs - 1) & ~63; i0 >= 0; i0 -= 64) {  // the first 64 come last and stay
      look(i0);
      items += wave_add((float)tiles);
      total += wave_add((float)tiles * (float)s.len);
    }
    it.slice = paged_slice(items * (float)heads, total * (float)heads, p.target);
  }
  int before = 0, before_cut = 0, before_sliced = 0;
  int splits = 1;
  unsigned long long cuts = 0;  // which of the 64 sequences looked at are cut
  auto cut_up = [&] {
    splits = s.len <= it.slice ? 1 : (s.len + it.slice - 1) / it.slice;
    cuts = __ballot(splits > 1 && tiles > 0);
  };
  if (b.seqs <= 64) {
    if (p.target == 0) look(0);
    cut_up();
    if (CUT && cuts == 0) return it;
  }
  for (int part = 0, i0 = 0; part < PARTS; i0 + 64 < b.seqs ? i0 += 64 : (i0 = 0, ++part)) {
    if (b.seqs > 64) {
      look(i0);
      cut_up();
    }
    const int behind = PARTS == 1 ? 0 : (int)((long long)tiles * part / PARTS);  // tiles of the parts before
    const int here = PARTS == 1 ? tiles : (int)((long long)tiles * (part + 1) / PARTS) - behind;
    // a cu_new that descends can count rows many times over: no sum of items passes the range of int
    const long long whole = (long long)here * heads, all = whole * splits;
    const int n = all > 0x800000 ? 0x800000 : (int)all;
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
  __device__ __forceinline__ PagedRows(const PagedItem& it, const PagedAttn& a, int G, int rows_per_tile) : group(G), step(a.q_heads) {
    const int first = it.tile * rows_per_tile, t0 = first / G;
    rest = first - t0 * G;
    out0 = (long long)(it.s.row0 + t0) * a.q_heads + it.head * G;
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

constexpr int PA_THREADS = PA_WAVES * 64;
// The slices of one item, COUNT of its ROWS rows from `first` on, by the threads of one workgroup.  A place is four
// columns of a row.  Its slices add up in four chains, every fourth slice to one, by four threads that meet in the LDS where
// places are few: the order, and the bits, are the same whoever joins.
constexpr int CHAINS = 4;
template <int ROWS, int COUNT, int DP, int OUT, bool THROUGH>
__device__ __forceinline__ void join_slices(const PagedAttn& a, const PagedCache& c, const PagedPlan& p, const PagedItem& it,
                                            float* meet, int first) {
  const int G = p.group, tid = threadIdx.x;
  const int live_rows = it.s.T * G - it.tile * ROWS - first;
  const int rows = COUNT < live_rows ? COUNT : live_rows;
  if (rows <= 0) return;
  constexpr int QUADS = DP / 4;  // places of a row; those beyond the head size are idle
  const int work = rows * QUADS;
  const float* tail = p.ws + (long long)p.places * ROWS * DP;
  const PagedRows out_row(it, a, G, ROWS);
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
    const int r = first + e / QUADS, d = e % QUADS * 4;
    if (d >= c.D) return;
    const float f = sum.den > 0.0f ? a.alpha_pv * 1024.0f / sum.den : 0.0f;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = sum.den > 0.0f ? sum.y[i] * f : 0.0f;
    store_some<4, OUT>(a.out, out_row(r) * c.D + d, y);
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
template <int ROWS, int DP, int OUT>
__device__ __forceinline__ void meet_and_join(const PagedAttn& a, const PagedCache& c, const PagedPlan& p, const PagedItem& it,
                                              int* seen, float* scratch) {
  if (p.arrivals == nullptr) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    seen[0] = __hip_atomic_fetch_add(p.arrivals + it.place, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (seen[0] == it.splits - 1) __hip_atomic_store(p.arrivals + it.place, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (seen[0] != it.splits - 1) return;
  join_slices<ROWS, ROWS, DP, OUT, true>(a, c, p, it, scratch, 0);
}

// Few rows: 16 to a workgroup, its four waves take 32 keys each in turn.  Bound by memory: 61 sequences of 40 to 4001 keys, 8 key
// heads of four query heads, 252 MB, take 57 us (4.4 TB/s; a copy of as much runs at 5.25), 2 x 95000 keys 389 MB in 70 us (5.6).
// A build that only loads takes as long; non-temporal loads, four waves to a SIMD instead of three and 64 keys a step did not help.
// Short sequences are a chain of latencies: 500 keys, 12 heads take 6.8 us, some 2 us of them to the first key.
constexpr int rows_lds(int DP) { return PA_WAVES * PA_ROWS * (DP + 4 + 2) * 4; }
template <int DP, int OUT>
__device__ __forceinline__ void paged_rows(const PagedAttn& a, const PagedCache& c, const PagedBatch& b, const PagedPlan& p, int index,
                                           char* lds) {
  constexpr int NB = DP / 16;    // column blocks; lane n of 16 owns the columns NB n .. NB n + NB - 1
  constexpr int KC = DP / 64;    // 16-byte pieces of a key row that a lane holds
  constexpr int VW = NB / 4;     // dwords of a value row that a lane holds
  const auto sum = reinterpret_cast<float(*)[PA_ROWS][DP + 4]>(lds);
  const auto offs = reinterpret_cast<float(*)[PA_ROWS]>(lds + PA_WAVES * PA_ROWS * (DP + 4) * 4);
  const auto den = offs + PA_WAVES;

  const PagedItem it = paged_item<1>(b, c.page_shift, c.heads, PA_ROWS, p, index);
  if (!it.found) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int G = p.group, live_rows = it.s.T * G;
  const int row = it.tile * PA_ROWS + n;              // of this lane's scores
  const int t = row / G, g = row - t * G;
  const int base = it.s.len - it.s.T;                 // position of the first new token (negative: it has none)
  const bool real = row < live_rows;
  int limit = real ? base + t + 1 : 0x7fffffff;       // keys of the row; rows that nobody asked for see what they like
  limit = limit < 0 ? 0 : limit;
  int last_row = it.tile * PA_ROWS + PA_ROWS - 1;
  last_row = last_row < live_rows - 1 ? last_row : live_rows - 1;
  int keys = base + last_row / G + 1;                 // keys of the last row: of the tile
  keys = keys < 0 ? 0 : keys;
  int first_limit = base + it.tile * PA_ROWS / G + 1; // keys of the first row
  const long long lo_ll = (long long)it.split * it.slice;
  const int lo = lo_ll < keys ? (int)lo_ll : keys;
  const int hi = lo_ll + it.slice < keys ? (int)(lo_ll + it.slice) : keys;

  // Q^T: 16 bytes a lane and MFMA; chunks beyond the head size are zeros, which add nothing
  v4i qf[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    qf[i] = v4i{0, 0, 0, 0};
    const int d = (i * 4 + kg) * 16;
    if (real && d < c.D)
      qf[i] = *reinterpret_cast<const v4i*>(a.q + (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head + d);
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const int8_t* kb = c.k + it.head * c.k_head;
  const int8_t* vb = c.v + it.head * c.v_head;
  // The table through the constant address space: nothing writes to it while the kernel runs, and scalar loads are counted
  // apart from the keys and values in flight, which a vector load would have to wait for.
  const auto table = (const __attribute__((address_space(4))) int*)(b.table + (long long)it.seq * b.per_seq);
  const int mask = (1 << c.page_shift) - 1, last_block = hi > 0 ? (hi - 1) >> 4 : 0;

  float off = PA_EMPTY;
  v4f acc[NB], dsum = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = v4f{0, 0, 0, 0};
  v8h ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (_Float16)1.0f;

  struct Step {
    v4i k[2][KC];
    unsigned v[8][VW];
    bool on[2];
  };
  // pages of the two blocks of 16 keys from s0 on, asked for a step before the keys are; blocks behind the last key are
  // masked, and read where there is memory
  auto pages_of = [&](int (&pg)[2], int s0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      int at = (s0 >> 4) + blk;
      at = at < last_block ? at : last_block;
      pg[blk] = table[(at << 4) >> c.page_shift];
    }
  };
  // Columns beyond the head size: the first ones are read instead, without a branch; Q is zero there, and what V makes of them
  // is not stored.
  unsigned kcol[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) kcol[i] = (unsigned)(n * c.k_token) + ((i * 4 + kg) * 16 < c.D ? (unsigned)(i * 4 + kg) * 16u : 0u);
  const unsigned vcol = (unsigned)(kg * 4 * c.v_token) + (n * NB < c.D ? (unsigned)(n * NB) : 0u);
  auto fetch = [&](Step& st, int s0, const int (&pg)[2]) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      int at = (s0 >> 4) + blk;
      at = at < last_block ? at : last_block;
      int page = pg[blk];
      st.on[blk] = page >= 0 && page < c.pages;
      page = st.on[blk] ? page : 0;
      const long long o = (at << 4) & mask;
      const int8_t* kr = kb + (long long)page * c.k_page + o * c.k_token;
#pragma unroll
      for (int i = 0; i < KC; ++i) st.k[blk][i] = *reinterpret_cast<const v4i*>(kr + kcol[i]);
      const int8_t* vr = vb + (long long)page * c.v_page + o * c.v_token;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VW == 2) {
          const v2u x = *reinterpret_cast<const v2u*>(vr + vcol);
          st.v[blk * 4 + j][0] = x[0];
          st.v[blk * 4 + j][1] = x[1];
        } else {
          st.v[blk * 4 + j][0] = *reinterpret_cast<const unsigned*>(vr + vcol);
        }
        vr += c.v_token;
      }
    }
  };
  auto work = [&](const Step& st, int s0) {
    float x[8];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      v4i s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KC; ++i) s = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.k[blk][i], qf[i], s, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[blk * 4 + r] = (float)s[r];
    }
    if (s0 + 32 > hi || s0 + 32 > first_limit || !st.on[0] || !st.on[1]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = s0 + (i >> 2) * 16 + kg * 4 + (i & 3);
        if (key >= hi || key >= limit || !st.on[i >> 2]) x[i] = -__builtin_inff();
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
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      unsigned u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = st.v[j][w] ^ 0x80808080u;  // v + 128, which is never negative
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // bytes of two rows as the low bytes of two fp16 numbers, (v + 128) 2^-24; times 2^14 less 2^-3 is v 2^-10, exactly
        v8h vf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned two = __builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x0c000c00u | (unsigned)(4 + i) << 16 | (unsigned)i);
          v2h h;
          __builtin_memcpy(&h, &two, 4);
          h = __builtin_elementwise_fma(h, v2h{(_Float16)16384.0f, (_Float16)16384.0f}, v2h{(_Float16)-0.125f, (_Float16)-0.125f});
          vf[2 * j] = h[0];
          vf[2 * j + 1] = h[1];
        }
        acc[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, hi_p, acc[4 * w + i], 0, 0, 0);
        acc[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, lo_p, acc[4 * w + i], 0, 0, 0);
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

  // the waves meet: lane (n, kg) holds of row n the columns NB (4 kg + r) + i in acc[i][r]
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < NB; i += 4)
      *reinterpret_cast<v4f*>(&sum[wave][n][NB * (4 * kg + r) + i]) = v4f{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
  if (kg == 0) {
    offs[wave][n] = off;
    den[wave][n] = dsum[0];
  }
  __syncthreads();
  const int quads = c.D / 4;
  const PagedRows out_row(it, a, G, PA_ROWS);
  for (int e = threadIdx.x; e < PA_ROWS * (DP / 4); e += PA_THREADS) {
    const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
    const int rr = it.tile * PA_ROWS + r;
    if (rr >= live_rows || d >= quads * 4) continue;
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
      const float f = l > 0.0f ? a.alpha_pv * 1024.0f / l : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = l > 0.0f ? y[i] * f : 0.0f;
      store_some<4, OUT>(a.out, out_row(r) * c.D + d, y);
    }
  }
  if (it.splits > 1) meet_and_join<PA_ROWS, DP, OUT>(a, c, p, it, reinterpret_cast<int*>(&offs[0][0]), &sum[0][0][0]);
}

// Many rows: 128 to a workgroup, 32 to each of its four waves, 64 keys to a step.  Each wave brings 16 of the keys: K as it is
// into rows of the LDS (16-byte chunks exchanged by the row, so that 32 rows are read without conflicts), V as fp16 in the order in
// which MFMA operands are read: of eight keys, chosen as S^T = K Q^T (32x32x32 int8) leaves them in a lane, one column in 16 bytes,
// lane after lane.  One widening of V then serves 128 rows.  Column blocks are interleaved (block i holds the columns NDB m + i),
// so a thread widens neighbouring columns and a lane of O^T ends up with neighbouring ones.
// Bound by what a wave can issue: a step of 64 keys takes a wave 1.6 us alone on its SIMD, the same with its keys in the nearest
// cache, and two waves 2.0 us (matrix pipe 38 % busy, vector ALUs 49 %; its 241 registers allow no third,
// but those of head sizes up to 64 do).  2048 rows over 16229 keys, 8 key heads of four: 442 to 456 us a pass, 510 G operations, half
// of them int8, half fp16.  An item costs 4 us before its first step
// (its place, its page, its keys) and some 2 behind the last: 4 x 512 rows of 40 heads are 640 items of 2 to 8 steps, 35 us.
// A probability is one fp16 number here, 11 bits: there is no time to spare that a second one could go into, as it does where few
// rows wait for memory.  With two (the sum of them in numerator and denominator, 255 registers) 2048 rows over 16229 keys take 657 us
// instead of 445, 512 rows beside 31 single tokens 47.6 instead of 41.0, 4 x 512 rows of 40 heads 38.4 instead of 34.3.  What that
// would gain, root mean square of the error over that of the contexts: 2.5e-4 to 2.1e-4 where contexts are fp16, whose own rounding
// is the 2.1e-4, and nothing to speak of in bf16 (1.7e-3).
// Scores start from 1.5 * 2^23 instead of 0: the int32 sum is then the fp32 number 12582912 + x, and the constant goes into the
// row's offset, where one multiply-add removes it exactly.
constexpr int PT_ROWS = 128, PT_KEYS = 64;
// Parts in which the tiles come (paged_item): 4 x 512 rows of 40 heads, four tiles to each, 39.1 us in one part, 38.3 in two, 36.5
// in four.
constexpr int PT_PARTS = 4;
constexpr int PT_JOIN = 32;      // rows that a workgroup joins
constexpr int PT_PLENTY = 2048;  // items from which on nothing is cut: four to each place on the chip
constexpr int tiles_lds(int DP) { return 3 * 3 * PT_KEYS * DP; }  // three steps of K, then of V as fp16
template <int DP, int OUT>
__device__ __forceinline__ void paged_tiles(const PagedAttn& a, const PagedCache& c, const PagedBatch& b, const PagedPlan& p, int index,
                                            char* lds) {
  constexpr int NDB = DP / 32;   // column blocks of O^T, and steps of 32 along a key row
  constexpr int KC = DP / 64;    // 16-byte pieces of K that a thread brings
  constexpr int CH = DP / 16;    // 16-byte chunks of a key row
  constexpr int KBYTES = PT_KEYS * DP, VBYTES = 2 * KBYTES;

  const PagedItem it = paged_item<PT_PARTS>(b, c.page_shift, c.heads, PT_ROWS, p, index);
  if (!it.found) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int G = p.group, live_rows = it.s.T * G;
  const int base = it.s.len - it.s.T;
  const int row0 = it.tile * PT_ROWS + wave * 32, row = row0 + n;
  const int t = row / G, g = row - t * G;
  const bool real = row < live_rows;
  int limit = real ? base + t + 1 : 0x7fffffff;
  limit = limit < 0 ? 0 : limit;
  const int first_limit = base + row0 / G + 1;   // keys of the wave's first row
  int keys = 0;                                  // keys of the wave's last row; none for a wave without rows
  if (row0 < live_rows) {
    const int last = row0 + 31 < live_rows ? row0 + 31 : live_rows - 1;
    keys = base + last / G + 1;
    keys = keys < 0 ? 0 : keys;
  }
  int most = it.tile * PT_ROWS + PT_ROWS - 1;    // keys of the workgroup's last row
  most = base + (most < live_rows ? most : live_rows - 1) / G + 1;
  most = most < 0 ? 0 : most;
  const long long lo_ll = (long long)it.split * it.slice;
  const int lo = lo_ll < most ? (int)lo_ll : most;
  const int hi = lo_ll + it.slice < most ? (int)(lo_ll + it.slice) : most;
  keys = keys < hi ? keys : hi;
  const int whole = first_limit < hi ? first_limit : hi;  // up to here every row of the wave sees every key

  v4i qf[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) {
    qf[i] = v4i{0, 0, 0, 0};
    const int d = i * 32 + h * 16;
    if (real && d < c.D)
      qf[i] = *reinterpret_cast<const v4i*>(a.q + (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head + d);
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const int8_t* kb = c.k + it.head * c.k_head;
  const int8_t* vb_ = c.v + it.head * c.v_head;
  const auto table = (const __attribute__((address_space(4))) int*)(b.table + (long long)it.seq * b.per_seq);
  const int mask = (1 << c.page_shift) - 1, last_block = hi > 0 ? (hi - 1) >> 4 : 0;

  // What this thread brings of a step: of the wave's 16 keys, KC chunks of K and the columns NDB n .. of eight rows of V.
  const int krow = lane / CH, kchunk = lane % CH;
  unsigned kcol[KC], vcol[8];
#pragma unroll
  for (int i = 0; i < KC; ++i) kcol[i] = (unsigned)((i * (64 / CH) + krow) * c.k_token) + (kchunk * 16 < c.D ? kchunk * 16u : 0u);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    vcol[j] = (unsigned)((h * 4 + (j & 3) + 8 * (j >> 2)) * c.v_token) + (n * NDB < c.D ? (unsigned)(n * NDB) : 0u);
  v4i kreg[KC];
  unsigned vreg[8];
  auto page_at = [&](int s0, int blk) {
    int at = (s0 >> 4) + blk;
    at = at < last_block ? at : last_block;
    return table[(at << 4) >> c.page_shift];
  };
  auto have = [&](int page) { return page >= 0 && page < c.pages; };
  auto place = [&](int s0) {  // where the wave's 16 keys begin in their page
    int at = (s0 >> 4) + wave;
    at = at < last_block ? at : last_block;
    return (at << 4) & mask;
  };
  auto k_from = [&](int s0, int page) { return kb + (long long)(have(page) ? page : 0) * c.k_page + place(s0) * c.k_token; };
  auto v_from = [&](int s0, int page) { return vb_ + (long long)(have(page) ? page : 0) * c.v_page + place(s0) * c.v_token; };
  // by buffer instructions: a column is one register beside the page's place in scalar ones, not two (241 registers instead of 255,
  // for head sizes up to 64 165 instead of 178, which makes room for a third workgroup: 16 x 512 rows of 32 heads 62.4 to 50.7 us)
  auto pool = [](const int8_t* from) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(from), 0, -1, 0x00020000); };
  auto fetch_k = [&](v4i (&kreg)[KC], const int8_t* from) {
    const auto r = pool(from);
#pragma unroll
    for (int i = 0; i < KC; ++i) kreg[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, kcol[i], 0, 0));
  };
  auto fetch_v = [&](unsigned (&vreg)[8], const int8_t* from) {
    const auto r = pool(from);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (NDB == 4) vreg[j] = __builtin_amdgcn_raw_buffer_load_b32(r, vcol[j], 0, 0);
      else vreg[j] = __builtin_amdgcn_raw_buffer_load_b16(r, vcol[j], 0, 0);
    }
  };
  auto swizzle = [](int r, int chunk) { return DP == 128 ? chunk ^ (r & 7) : chunk ^ ((r >> 2) & 3); };
  int kat[NDB];  // where this lane's operands of K begin, of the first 32 keys
#pragma unroll
  for (int i = 0; i < NDB; ++i) kat[i] = n * DP + swizzle(n, 2 * i + h) * 16;
  auto put_k = [&](const v4i (&kreg)[KC], int slot) {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const int r = wave * 16 + i * (64 / CH) + krow;
      *reinterpret_cast<v4i*>(lds + slot * KBYTES + r * DP + swizzle(r, kchunk) * 16) = kreg[i];
    }
  };
  // V: bytes plus 128 (which are never negative) as the low bytes of fp16 numbers, (v + 128) 2^-24; times 2^14 less 2^-3 is
  // v 2^-10, exactly
  unsigned vplus[8];
  auto lift = [&](int j) { vplus[j] = vreg[j] ^ 0x80808080u; };
  auto put_v = [&](int slot, int i) {
    v8h x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned two = __builtin_amdgcn_perm(vplus[2 * j + 1], vplus[2 * j], 0x0c000c00u | (unsigned)(4 + i) << 16 | (unsigned)i);
      v2h y;
      __builtin_memcpy(&y, &two, 4);
      y = __builtin_elementwise_fma(y, v2h{(_Float16)16384.0f, (_Float16)16384.0f}, v2h{(_Float16)-0.125f, (_Float16)-0.125f});
      x[2 * j] = y[0];
      x[2 * j + 1] = y[1];
    }
    *reinterpret_cast<v8h*>(lds + 3 * KBYTES + slot * VBYTES + ((wave * NDB + i) * 64 + lane) * 16) = x;
  };

  float off = PA_EMPTY, den = 0.0f;
  v16f acc[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
  v16i start;
#pragma unroll
  for (int r = 0; r < 16; ++r) start[r] = 0x4b400000;
  asm("" : "+v"(start));   // kept in registers, not made anew at every step

  // The operands of 32 keys: of K for their scores, of V for their products, first 16 keys and second.
  v4i kf[NDB];
  v8h va[NDB], vb[NDB];
  auto read_k = [&](int at, int i) { kf[i] = *reinterpret_cast<const v4i*>(lds + at + kat[i]); };
  auto read_v = [&](v8h (&v)[NDB], int at, int q, int i) { v[i] = *reinterpret_cast<const v8h*>(lds + at + ((q * NDB + i) * 64 + lane) * 16); };
  struct Half {
    v16f x;         // scores of 32 keys
    float top;      // the largest of them
    v8h pr[2];      // their probabilities
  };
  constexpr int BUNDLES = 3 * NDB;
  // 32 keys from s0 on: the softmax of their scores into their probabilities, beside it the scores of the next 32 keys and the
  // products of the 32 before, in bundles that the compiler keeps in order: a matrix instruction, then what runs beside
  // it.  A pair of scores goes through its multiply-adds and exponentials in one bundle, is rounded in the next and added to
  // the denominator in the one behind that, so nothing waits for the instruction before it; operands are read from the LDS
  // bundles, or a half, before they are used: kf and va are here, vb comes from `v_at`, the next half's from `k_next` and
  // `v_next`.  `beside(m)` is what else is to be done in bundle m.
  auto half = [&](Half& now, Half& next, v8h (&before)[2], int s0, int lost, int v_at, int k_next, int v_next, auto beside) {
    if (__builtin_expect(s0 + 32 > whole || lost != 0, 0)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = s0 + (r & 3) + 8 * (r >> 2) + 4 * h;
        if (key >= hi || key >= limit || (lost >> (r >> 3) & 1)) now.x[r] = -__builtin_inff();
      }
      now.top = now.x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) now.top = __builtin_fmaxf(now.top, now.x[r]);
    }
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
      const _Float16 scale_h = (_Float16)scale;
#pragma unroll
      for (int q = 0; q < 2; ++q) before[q] *= scale_h;
#pragma unroll
      for (int i = 0; i < NDB; ++i) acc[i] *= scale;
    }
    v16i t = start;
    v16f tf;
    float e[2][2];
    v2h two[8];
    auto softmax = [&](int m) {
      if (m >= 2 && m < 10) den = __builtin_amdgcn_fdot2(two[m - 2], v2h{(_Float16)1.0f, (_Float16)1.0f}, den, false);
      if (m >= 1 && m < 9) {
        two[m - 1] = v2h{(_Float16)e[(m - 1) & 1][0], (_Float16)e[(m - 1) & 1][1]};
        asm volatile("" : "+v"(two[m - 1]));  // computed here, not where the next half needs it
      }
      if (m < 8) {
        e[m & 1][0] = __builtin_amdgcn_exp2f(__builtin_fmaf(now.x[2 * m], cl, off));
        e[m & 1][1] = __builtin_amdgcn_exp2f(__builtin_fmaf(now.x[2 * m + 1], cl, off));
      }
    };
    __builtin_amdgcn_sched_barrier(0);
    softmax(0);
#pragma unroll
    for (int m = 0; m < BUNDLES; ++m) {
      __builtin_amdgcn_sched_barrier(0);
      const int i = m < 2 * NDB ? m >> 1 : m - 2 * NDB;
      if (m < 2 * NDB && (m & 1) == 0) t = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[i], qf[i], t, 0, 0, 0);
      else if (m < 2 * NDB) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[i], before[0], acc[i], 0, 0, 0);
      else acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb[i], before[1], acc[i], 0, 0, 0);
      softmax(m + 1);
      if (m < NDB) read_v(vb, v_at, 1, m);
      if (m >= 2 * NDB) {
        read_k(k_next, i);
        read_v(va, v_next, 0, i);
      }
      constexpr int PARTS = NDB == 4 ? 3 : 2;  // bundles at the end, in which the next scores are there
      const int part = m - (BUNDLES - PARTS);
      if (part == 0) __builtin_memcpy(&tf, &t, sizeof(t));
      if (part >= 0) {
#pragma unroll
        for (int r = 16 * part / PARTS; r < 16 * (part + 1) / PARTS; ++r) next.top = r == 0 ? tf[0] : __builtin_fmaxf(next.top, tf[r]);
      }
      beside(m);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = BUNDLES + 1; m < 10; ++m) softmax(m);
    asm volatile("" : "+v"(den), "+v"(next.top));
    next.x = tf;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        now.pr[q][2 * j] = two[q * 4 + j][0];
        now.pr[q][2 * j + 1] = two[q * 4 + j][1];
      }
  };

  if (lo < hi) {
    // Pages are looked up a step ahead, by vector loads: these return in order, so that the wait for the keys and values in
    // front of one is all the wait it needs (a scalar one would have to be over at every wait for the LDS).
    int zero = 0;
    asm("" : "+v"(zero));
    auto ask = [&](int s0) {
      int at = (s0 >> 4) + wave;
      at = at < last_block ? at : last_block;
      return b.table[(long long)it.seq * b.per_seq + ((at << 4) >> c.page_shift) + zero];
    };
    // the first three steps of K and two of V are asked for at once
    const int page0 = page_at(lo, wave), page1 = page_at(lo + PT_KEYS, wave);
    int page_v = page_at(lo + 2 * PT_KEYS, wave);
    int asked = ask(lo + 3 * PT_KEYS);
    v4i k_0[KC], k_1[KC];
    unsigned v_0[8];
    fetch_k(k_0, k_from(lo, page0));
    fetch_v(v_0, v_from(lo, page0));
    fetch_k(k_1, k_from(lo + PT_KEYS, page1));
    fetch_v(vreg, v_from(lo + PT_KEYS, page1));
    fetch_k(kreg, k_from(lo + 2 * PT_KEYS, page_v));
    // whether the pool lacks any of the item's pages: looked at once, while the first keys are on their way, so that steps need not
    bool holes = false;
    for (int i = (lo >> c.page_shift) + lane; i <= (hi - 1) >> c.page_shift; i += 64) holes |= !have(table[i]);
    holes = __ballot(holes) != 0;
    auto lost = [&](int s0) {
      int bits = 0;
      if (__builtin_expect(holes, 0))
        for (int i = 0; i < 4; ++i) bits |= (have(page_at(s0, i)) ? 0 : 1) << i;
      return bits;
    };
    put_k(k_0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) vplus[j] = v_0[j] ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < NDB; ++i) put_v(0, i);
    put_k(k_1, 1);
    __syncthreads();
    constexpr int V0 = 3 * KBYTES, K_HALF = 32 * DP, V_HALF = VBYTES / 2;
    Half even, odd;
    {
#pragma unroll
      for (int i = 0; i < NDB; ++i) read_k(0, i);
      v16i t = start;
#pragma unroll
      for (int i = 0; i < NDB; ++i) t = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[i], qf[i], t, 0, 0, 0);
      __builtin_memcpy(&even.x, &t, sizeof(t));
      even.top = even.x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) even.top = __builtin_fmaxf(even.top, even.x[r]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) odd.pr[q][j] = (_Float16)0.0f;
    // slots of this step, of the next one and of the one behind it; V of the step before is in the third of them
    int k0 = 0, k1 = 1, k2 = 2;
    int v_before = V0 + V_HALF;   // (the first step takes its own V, times zero)
#pragma unroll
    for (int i = 0; i < NDB; ++i) {
      read_k(K_HALF, i);
      read_v(va, v_before, 0, i);
    }
    // A step is 64 keys.  What is read in it: the second half of its K and the first of the next one's, the second half of V
    // before it and the first of its own, and ahead of the next step K's second half of that and V's of this; what is written:
    // V of the next step and K of the one behind that, in places that the step before has read, which one barrier a step
    // makes sure of.
    int s0 = lo;
    for (;;) {
      const int gone = lost(s0);
      // the same for all lanes: with the half behind its last keys a wave gathers those
      const bool here = __builtin_amdgcn_readfirstlane(s0 < keys + 32) != 0;
      const int v_now = V0 + k0 * VBYTES;
      const int8_t* from;
      auto stage_v = [&](int m) {
        if (m == 0) from = v_from(s0 + 2 * PT_KEYS, page_v);
        if (m >= NDB && m < 2 * NDB) {
#pragma unroll
          for (int j = 0; j < 8 / NDB; ++j) lift((m - NDB) * (8 / NDB) + j);
        }
        if (m == 2 * NDB) fetch_v(vreg, from);
        if (m >= 2 * NDB) put_v(k1, m - 2 * NDB);
      };
      auto stage_k = [&](int m) {
        if (m == 0) {
          page_v = __builtin_amdgcn_readfirstlane(asked);
          from = k_from(s0 + 3 * PT_KEYS, page_v);
        }
        if (m == NDB) put_k(kreg, k2);
        if (m == NDB + 1) {
          fetch_k(kreg, from);
          asked = ask(s0 + 4 * PT_KEYS);
        }
      };
      if (__builtin_expect(here, 1)) {
        half(even, odd, odd.pr, s0, gone & 3, v_before, k1 * KBYTES, v_now, stage_v);
        half(odd, even, even.pr, s0 + 32, gone >> 2, v_now, k1 * KBYTES + K_HALF, v_now + V_HALF, stage_k);
      } else {
#pragma unroll
        for (int m = 0; m < BUNDLES; ++m) stage_v(m);
#pragma unroll
        for (int m = 0; m < BUNDLES; ++m) stage_k(m);
        // nothing is left on its way into registers that the other path uses for something else: it would wait for all its loads
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      }
      __syncthreads();
      v_before = v_now + V_HALF;
      const int k = k0;
      k0 = k1, k1 = k2, k2 = k;
      s0 += PT_KEYS;
      if (s0 >= hi) break;
    }
    if (s0 < keys + 32) {  // nobody has gathered them: the wave's keys reach into the last half
#pragma unroll
      for (int i = 0; i < NDB; ++i) read_v(vb, v_before, 1, i);
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[i], odd.pr[0], acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb[i], odd.pr[1], acc[i], 0, 0, 0);
      }
    }
  }

  // a lane has its row's columns NDB m + i, m = (r & 3) + 8 (r >> 2) + 4 h; the two halves of the wave add their denominators
  {
    auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(den), __float_as_uint(den), false, false);
    den = __uint_as_float(o[0]) + __uint_as_float(o[1]);
  }
  // Through the LDS, four columns at a place that the row moves, so that rows leave as whole lines.
  __syncthreads();
  float f = 1.0f;
  if (it.splits == 1) f = den > 0.0f ? a.alpha_pv * 1024.0f / den : 0.0f;
  constexpr int QUADS = DP / 4, PER = 64 / QUADS;  // rows that a wave stores at once
  v4f* const own = reinterpret_cast<v4f*>(lds) + wave * 32 * QUADS;
  auto spot = [](int r, int quad) { return r * QUADS + (quad ^ (r & (QUADS - 1))); };
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = (r & 3) + 8 * (r >> 2) + 4 * h;
    float y[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i) y[i] = f > 0.0f || f < 0.0f ? acc[i][r] * f : 0.0f;
    if constexpr (NDB == 4) own[spot(n, m)] = v4f{y[0], y[1], y[2], y[3]};
    else *(reinterpret_cast<v2f*>(&own[spot(n, m >> 1)]) + (m & 1)) = v2f{y[0], y[1]};
  }
  __builtin_amdgcn_wave_barrier();
  const long long slot = it.place + (long long)it.split * it.step;
  const int quad = lane % QUADS;
  const PagedRows out_row(it, a, G, PT_ROWS);
#pragma unroll
  for (int i = 0; i < 32 / PER; ++i) {
    const int r = i * PER + lane / QUADS, rr = row0 + r;
    if (rr >= live_rows || quad * 4 >= c.D) continue;
    const v4f y = own[spot(r, quad)];
    if (it.splits == 1) {
      store_some<4, OUT>(a.out, out_row(wave * 32 + r) * c.D + quad * 4, {y[0], y[1], y[2], y[3]});
    } else {
      *reinterpret_cast<v4f*>(p.ws + (slot * PT_ROWS + wave * 32 + r) * DP + quad * 4) = v4f{y[0], y[1], y[2], y[3]};
    }
  }
  if (it.splits > 1 && real && h == 0)
    *reinterpret_cast<v2f*>(p.ws + (long long)p.places * PT_ROWS * DP + (slot * PT_ROWS + wave * 32 + n) * 2) = v2f{off, den};
}

template <int DP, int OUT>
__global__ __launch_bounds__(PA_THREADS, 3) void paged_attn_rows_kernel(PagedAttn a, PagedCache c, PagedBatch b, PagedPlan rows) {
  __shared__ __attribute__((aligned(16))) char lds[rows_lds(DP)];
  const int lo = b.cu[0], hi = b.cu[b.seqs];  // (on their way beside what the item needs)
  paged_rows<DP, OUT>(a, c, b, rows, blockIdx.x, lds);
  if (a.fill) paged_fill(b, lo, hi, static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
}

// Sequences of few rows and of many in one launch, 256 items of the one kind after 256 of the other as long as both last: those
// with few rows wait for memory while the others compute.  Workgroups go in turn to the eight XCDs, within one to its four shader
// engines, within one to its eight CUs, and the next waits until there is room at its own engine: so 256 leave one of each kind
// to every CU, while turns of 1, 8 or 32 leave the long items, two to a CU, to half of the chip, with the other half idle
// behind them (512 rows over 2000 keys beside a sequence of one row: 56.7 us by 8, 45.4 by 32, 39.5 by 256).
constexpr int TURN = 256;
template <int DP, int OUT>
__global__ __launch_bounds__(PA_THREADS, DP == 64 ? 3 : 2) void paged_attn_both_kernel(PagedAttn a, PagedCache c, PagedBatch b, PagedPlan rows,
                                                                        PagedPlan tiles) {
  __shared__ __attribute__((aligned(16))) char lds[tiles_lds(DP) > rows_lds(DP) ? tiles_lds(DP) : rows_lds(DP)];
  if (a.fill) paged_fill(b, b.cu[0], b.cu[b.seqs], static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
  const int i = blockIdx.x, each = (rows.slots < tiles.slots ? rows.slots : tiles.slots) & -TURN, rest = i - 2 * each;
  const bool many = rest < 0 ? (i & TURN) == 0 : rest < tiles.slots - each;
  const int index = rest < 0 ? i / (2 * TURN) * TURN + i % TURN : each + rest - (many ? 0 : tiles.slots - each);
  if (many) paged_tiles<DP, OUT>(a, c, b, tiles, index, lds);
  else paged_rows<DP, OUT>(a, c, b, rows, index, lds);
}

// Joins slices that do not meet in the launch itself: an item that was cut to ROWS / EACH workgroups, EACH of its rows to one.
// Eight items take turns, so that what there is to join comes first and goes to all CUs, and that an item whose number leaves the
// same rest by 8 as its slices' (as where key heads come in eights) is read by the XCD that has written it.
template <int ROWS, int EACH, int DP, int OUT>
__global__ __launch_bounds__(PA_THREADS) void paged_attn_join_kernel(PagedAttn a, PagedCache c, PagedBatch b, PagedPlan p) {
  __shared__ __attribute__((aligned(16))) float meet[PA_THREADS * 8];
  constexpr int PIECES = ROWS / EACH;
  const PagedItem it = paged_item<ROWS == PT_ROWS ? PT_PARTS : 1, true>(b, c.page_shift, c.heads, ROWS, p,
                                                                                 blockIdx.x / (8 * PIECES) * 8 + blockIdx.x % 8);
  if (!it.found || it.split != 0) return;
  join_slices<ROWS, EACH, DP, OUT, false>(a, c, p, it, meet, blockIdx.x / 8 % PIECES * EACH);
}

// What a call of these sizes runs.  The lengths are on the device, so the grids and the workspace are bounds.  The grid: one item to
// each (sequence, key head, tile of rows) and the slices beyond that.  The workspace: an item that is cut is longer than a slice,
// a slice at least the target-th part of all keys, so there are fewer than `target` such items, and of their slices fewer than
// `target` whole ones and one more to each.
struct PagedShape {
  long long rows_slots, tiles_slots;    // items of either kind, slices included; 0: none
  long long rows_places, tiles_places;  // slices of those that are cut
  int rows_target, tiles_target;        // slices that the keys are cut into; 0: nothing is cut
  bool rows_meet;                       // slices of few rows meet in the launch
  static long long places(long long slots, int target) { return slots < 2 * target + 8 ? slots : 2 * target + 8; }
  void cut_rows(int target, long long each) {
    rows_target = target;
    // where the slices of an item come to more than 65 KB, one workgroup would be longer in joining them than another launch
    // takes (2 x 100000 keys, 8 key heads of 8: 135 KB, 87 us in all against 71.6 + 5.5 us)
    rows_meet = target * each * 520 <= 66560 * rows_slots;
    rows_slots += target + 8;
    rows_places = places(rows_slots, target);
  }
  void cut_tiles(int target) {
    tiles_target = target;
    tiles_slots += target + 8;
    tiles_places = places(tiles_slots, target);
  }
};
static PagedShape paged_shape(long long rows, long long seqs, long long group, long long heads, long long capacity) {
  PagedShape s = {0, 0, 0, 0, 0, 0, false};
  const bool cut = seqs > 0 && capacity > PA_MIN_SLICE;
  if (rows * group <= PA_ROWS * seqs) {  // few rows to a sequence on average: all of them by that kernel
    s.rows_slots = heads * (seqs + rows * group / PA_ROWS);
    const long long each = rows * group / seqs + 1 < PA_ROWS ? rows * group / seqs + 1 : PA_ROWS;
    if (cut) s.cut_rows(PA_TARGET, each);
    return s;
  }
  // sequences with more than 16 rows are at most a 17th of all rows
  const long long many = rows * group / (PA_ROWS + 1) < seqs ? rows * group / (PA_ROWS + 1) : seqs;
  s.tiles_slots = heads * (many + rows * group / PT_ROWS);
  const bool cut_tiles = cut && s.tiles_slots < PT_PLENTY;
  if (seqs == 1) {  // it has more than 16
    if (cut_tiles) s.cut_tiles(PA_TARGET);
    return s;
  }
  // Where both kinds share the chip, a place on each CU for the tiles, and few cuts for the others, which have the time: 512 rows over
  // 600 to 2007 keys beside 31 sequences of one row took 58.8 us with 512 slices of each kind, 48.3 with 256 of each, 44.4 with
  // 256 of tiles and 128 of the others.
  s.rows_slots = heads * seqs;
  if (cut_tiles) s.cut_tiles(PA_TARGET / 2);
  if (cut) s.cut_rows(PA_TARGET / 4, PA_ROWS);
  return s;
}
static int paged_dp(long long D) { return D <= 64 ? 64 : 128; }
static long long paged_bytes(long long places, int rows, long long D) { return places * rows * (paged_dp(D) + 2) * 4; }

long long paged_attn_arrivals(long long rows, long long seqs, long long q_heads, long long heads, long long capacity) {
  const PagedShape s = paged_shape(rows, seqs, q_heads / heads, heads, capacity);
  return s.rows_meet ? s.rows_places : 0;
}
long long paged_attn_workspace_bytes(long long rows, long long seqs, long long q_heads, long long heads, long long D,
                                     long long capacity) {
  const PagedShape s = paged_shape(rows, seqs, q_heads / heads, heads, capacity);
  return (s.rows_target ? paged_bytes(s.rows_places, PA_ROWS, D) : 0) + (s.tiles_target ? paged_bytes(s.tiles_places, PT_ROWS, D) : 0);
}

template <int DP, int OUT>
static void launch_attn(const PagedAttn& a, const PagedCache& c, const PagedBatch& b, const PagedPlan& rows, const PagedPlan& tiles,
                        hipStream_t stream) {
  const unsigned grid = (unsigned)(rows.slots + tiles.slots > 0 ? rows.slots + tiles.slots : 1);
  if (tiles.slots > 0)
    hipLaunchKernelGGL((paged_attn_both_kernel<DP, OUT>), dim3(grid), dim3(PA_THREADS), 0, stream, a, c, b, rows, tiles);
  else
    hipLaunchKernelGGL((paged_attn_rows_kernel<DP, OUT>), dim3(grid), dim3(PA_THREADS), 0, stream, a, c, b, rows);
  // an item that is cut has more than a target-th of all keys, so there are fewer than `target` of them
  auto items = [](const PagedPlan& p) {
    const int most = p.slots - p.target - 8;
    return (unsigned)((most < p.target ? most : p.target) + 7 & ~7);
  };
  if (rows.target > 0 && rows.arrivals == nullptr)
    hipLaunchKernelGGL((paged_attn_join_kernel<PA_ROWS, 2, DP, OUT>), dim3(items(rows) * (PA_ROWS / 2)), dim3(PA_THREADS), 0,
                       stream, a, c, b, rows);
  if (tiles.target > 0)
    hipLaunchKernelGGL((paged_attn_join_kernel<PT_ROWS, PT_JOIN, DP, OUT>), dim3(items(tiles) * (PT_ROWS / PT_JOIN)), dim3(PA_THREADS),
                       0, stream, a, c, b, tiles);
}

int launch_paged_attn_s8(int out_type, const PagedAttn& a, const PagedCache& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream) {
  if (b.rows == 0 || a.q_heads == 0) return TI_OK;
  const int group = a.q_heads / c.heads;
  const long long capacity = (long long)b.per_seq << c.page_shift;
  PagedShape s = paged_shape(b.rows, b.seqs, group, c.heads, capacity);
  if (workspace == nullptr || workspace_bytes < paged_attn_workspace_bytes(b.rows, b.seqs, a.q_heads, c.heads, c.D, capacity))
    s.rows_target = s.tiles_target = 0, s.rows_meet = false;
  if (s.rows_slots + s.tiles_slots > 0x7fffff)
    return fail(TI_ERR_INVALID_ARG, "paged_attn_s8: %lld work items", s.rows_slots + s.tiles_slots);
  const bool meet = a.arrivals != nullptr && a.arrivals_count >= paged_attn_arrivals(b.rows, b.seqs, a.q_heads, c.heads, capacity);
  char* ws = static_cast<char*>(workspace);
  PagedPlan rows, tiles;
  rows.group = tiles.group = group;
  rows.least = 0;
  rows.most = s.tiles_slots > 0 ? PA_ROWS : 0x7fffffff;
  rows.slots = (int)s.rows_slots;
  rows.places = (int)s.rows_places;
  rows.target = s.rows_target;
  rows.ws = reinterpret_cast<float*>(ws);
  rows.arrivals = meet && s.rows_meet ? a.arrivals : nullptr;
  tiles.least = s.rows_slots > 0 ? PA_ROWS : 0;
  tiles.most = 0x7fffffff;
  tiles.slots = (int)s.tiles_slots;
  tiles.places = (int)s.tiles_places;
  tiles.target = s.tiles_target;
  tiles.ws = reinterpret_cast<float*>(ws + (s.rows_target ? paged_bytes(s.rows_places, PA_ROWS, c.D) : 0));
  tiles.arrivals = nullptr;  // slices of 66 KB: many workgroups join them, in a launch of their own
  auto run = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (out_type == PT_S8) launch_attn<DP, PT_S8>(a, c, b, rows, tiles, stream);
    else if (out_type == PT_F16) launch_attn<DP, PT_F16>(a, c, b, rows, tiles, stream);
    else launch_attn<DP, PT_BF16>(a, c, b, rows, tiles, stream);
  };
  if (paged_dp(c.D) == 64) run(std::integral_constant<int, 64>());
  else run(std::integral_constant<int, 128>());
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_attn_s8 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

}  // namespace ti
