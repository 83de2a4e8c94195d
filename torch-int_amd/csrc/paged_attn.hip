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

constexpr int PA_WAVES = 8;
constexpr int PA_ROWS = 16;
constexpr int PA_TARGET = 1024;    // work items that the keys are cut into, beyond one to each (sequence, key head, 16 rows)
constexpr int PA_MIN_SLICE = 512;  // keys of a slice, at least
constexpr float PA_EMPTY = 3.0e38f;  // offset of a row that has seen no key: 2^(-inf + PA_EMPTY) is 0

struct PagedPlan {
  int group;      // query heads of a key head
  int target;     // slices beyond which nothing is cut; 0: nothing is cut at all
  int slots;      // items the workspace holds
};

struct PagedItem {
  PagedSeq s;
  int seq, head, tile, split, splits, first;  // `first`: slot of the item's slice 0 (its slices are kv_heads * tiles apart)
  int step;                                   // slots from one slice to the next
  int slice;                                  // keys of a slice
  bool found;
};

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = v + __shfl_xor(v, off, 64);
  return v;
}

// Keys of a slice, the same in every workgroup: what cuts all keys of the batch into `target` equal parts.
__device__ __forceinline__ int paged_slice(const PagedBatch& b, int page_shift, int heads, int rows_per_tile, const PagedPlan& p) {
  if (p.target == 0) return 0x7fffffff;
  const int lane = threadIdx.x & 63;
  float total = 0.0f;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    float mine = 0.0f;
    if (i0 + lane < b.seqs) {
      const PagedSeq s = paged_seq(b, page_shift, i0 + lane);
      mine = (float)((s.T * p.group + rows_per_tile - 1) / rows_per_tile) * (float)s.len;
    }
    total += wave_add(mine);
  }
  const float want = total * (float)heads / (float)p.target;
  int slice = want < 1.0e9f ? ((int)want + 64) & ~63 : 1 << 30;
  return slice < PA_MIN_SLICE ? PA_MIN_SLICE : slice;
}

// The work item with number `index`, in the order sequence, slice, tile of rows, head.
__device__ __forceinline__ PagedItem paged_item(const PagedBatch& b, int page_shift, int heads, int rows_per_tile, const PagedPlan& p,
                                                int index) {
  PagedItem it;
  it.found = false;
  it.slice = paged_slice(b, page_shift, heads, rows_per_tile, p);
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    PagedSeq s = {0, 0, 0};
    int n = 0, tiles = 0, splits = 0;
    if (i0 + lane < b.seqs) {
      s = paged_seq(b, page_shift, i0 + lane);
      tiles = (s.T * p.group + rows_per_tile - 1) / rows_per_tile;
      splits = s.len <= it.slice ? 1 : (s.len + it.slice - 1) / it.slice;
      n = tiles * splits * heads;
    }
    int upto = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(upto, off, 64);
      if (lane >= off) upto += o;
    }
    const unsigned long long past = __ballot(before + upto > index);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int first = before + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at);
      const int rel = index - first;
      const int t = __builtin_amdgcn_readlane(tiles, at);
      it.s.row0 = __builtin_amdgcn_readlane(s.row0, at);
      it.s.T = __builtin_amdgcn_readlane(s.T, at);
      it.s.len = __builtin_amdgcn_readlane(s.len, at);
      it.splits = __builtin_amdgcn_readlane(splits, at);
      it.seq = i0 + at;
      it.step = heads * t;
      it.split = rel / it.step;
      const int rest = rel - it.split * it.step;
      it.tile = rest / heads;
      it.head = rest - it.tile * heads;
      it.first = first + rest;
      // cu_new that does not ascend can count rows twice, and with them items past the range of int: no item then
      it.found = first >= 0 && rel >= 0 && it.split < it.splits && it.tile < t;
      return it;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return it;
}

// Rows of no sequence (behind the last one; in front of the first, should it not begin at row 0) become zeros.
__device__ __forceinline__ void paged_fill(const PagedBatch& b, char* out, long long row_bytes) {
  int lo = b.cu[0], hi = b.cu[b.seqs];
  lo = lo < 0 ? 0 : lo > b.rows ? b.rows : lo;
  hi = hi < lo ? lo : hi > b.rows ? b.rows : hi;
  const int rest = b.rows - (hi - lo);
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    char* at = out + (long long)(i < lo ? i : hi + i - lo) * row_bytes;
    for (long long j = threadIdx.x * 16ll; j < row_bytes; j += blockDim.x * 16ll) *reinterpret_cast<v4i*>(at + j) = v4i{0, 0, 0, 0};
  }
}

template <int OUT>
__device__ __forceinline__ void store4(void* out, long long at, const float (&y)[4]) {
  if constexpr (OUT == PT_S8) {
    int w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (rne_s8(y[i]) & 255) << (8 * i);
    reinterpret_cast<int*>(static_cast<int8_t*>(out) + at)[0] = w;
  } else {
    unsigned short h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (OUT == PT_F16) {
        const _Float16 v = (_Float16)y[i];
        __builtin_memcpy(&h[i], &v, 2);
      } else {
        const __bf16 v = (__bf16)y[i];
        __builtin_memcpy(&h[i], &v, 2);
      }
    }
    int2 w;
    __builtin_memcpy(&w, h, 8);
    *reinterpret_cast<int2*>(static_cast<unsigned short*>(out) + at) = w;
  }
}

// Workspace: partial sums [slots][16][DP] fp32, then offsets [slots][16] and denominators [slots][16].
template <int DP, int OUT>
__global__ __launch_bounds__(PA_WAVES * 64) void paged_attn_rows_kernel(PagedAttn a, PagedCache c, PagedBatch b, PagedPlan p,
                                                                        float* ws) {
  constexpr int NB = DP / 16;    // column blocks; lane n of 16 owns the columns NB n .. NB n + NB - 1
  constexpr int KC = DP / 64;    // 16-byte pieces of a key row that a lane holds
  constexpr int VW = NB / 4;     // dwords of a value row that a lane holds
  __shared__ __attribute__((aligned(16))) float sum[PA_WAVES][PA_ROWS][DP + 4];
  __shared__ float offs[PA_WAVES][PA_ROWS], den[PA_WAVES][PA_ROWS];

  if (a.fill) paged_fill(b, static_cast<char*>(a.out), (long long)a.q_heads * c.D * (OUT == PT_S8 ? 1 : 2));
  const PagedItem it = paged_item(b, c.page_shift, c.heads, PA_ROWS, p, blockIdx.x);
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
    const int d = (kg * KC + i) * 16;
    if (real && d < c.D)
      qf[i] = *reinterpret_cast<const v4i*>(a.q + (long long)(it.s.row0 + t) * a.q_row + (long long)(it.head * G + g) * a.q_head + d);
  }
  const float cl = a.alpha_qk * 1.44269504088896341f;
  const int8_t* kb = c.k + it.head * c.k_head;
  const int8_t* vb = c.v + it.head * c.v_head;
  const int* table = b.table + (long long)it.seq * b.per_seq;
  const int mask = (1 << c.page_shift) - 1, last_block = keys > 0 ? (keys - 1) >> 4 : 0;

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
  auto fetch = [&](Step& st, int s0) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      int at = (s0 >> 4) + blk;
      at = at < last_block ? at : last_block;  // blocks behind the last key: masked, read where there is memory
      int page = table[(at << 4) >> c.page_shift];
      st.on[blk] = page >= 0 && page < c.pages;
      page = st.on[blk] ? page : 0;
      const int o = (at << 4) & mask;
      const int8_t* kr = kb + (long long)page * c.k_page + (long long)(o + n) * c.k_token;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const int d = (kg * KC + i) * 16;
        st.k[blk][i] = v4i{0, 0, 0, 0};
        if (d < c.D) st.k[blk][i] = *reinterpret_cast<const v4i*>(kr + d);
      }
      const int8_t* vr = vb + (long long)page * c.v_page + (long long)(o + kg * 4) * c.v_token + n * NB;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int w = 0; w < VW; ++w) st.v[blk * 4 + j][w] = 0;
        if (n * NB < c.D) {
          if constexpr (VW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(vr + (long long)j * c.v_token);
            st.v[blk * 4 + j][0] = x.x;
            st.v[blk * 4 + j][1] = x.y;
          } else {
            st.v[blk * 4 + j][0] = *reinterpret_cast<const unsigned*>(vr + (long long)j * c.v_token);
          }
        }
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
      float o = __shfl_xor(top, 16, 64);
      top = o > top ? o : top;
      o = __shfl_xor(top, 32, 64);
      top = o > top ? o : top;
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
    Step st;
    fetch(st, s0);
    for (;;) {
      const int next = s0 + PA_WAVES * 32;
      if (next >= hi) break;
      Step after;
      fetch(after, next);
      work(st, s0);
      st = after;
      s0 = next;
    }
    work(st, s0);
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
  for (int e = threadIdx.x; e < PA_ROWS * (DP / 4); e += PA_WAVES * 64) {
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
      const long long slot = it.first + (long long)it.split * it.step;
      if (slot >= p.slots) continue;
      *reinterpret_cast<v4f*>(ws + (slot * PA_ROWS + r) * DP + d) = v4f{y[0], y[1], y[2], y[3]};
      if (d == 0) {
        float* tail = ws + (long long)p.slots * PA_ROWS * DP;
        tail[slot * PA_ROWS + r] = least;
        tail[(long long)p.slots * PA_ROWS + slot * PA_ROWS + r] = l;
      }
    } else {
      const float f = l > 0.0f ? a.alpha_pv * 1024.0f / l : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = l > 0.0f ? y[i] * f : 0.0f;
      const int tt = rr / G;
      store4<OUT>(a.out, ((long long)(it.s.row0 + tt) * a.q_heads + it.head * G + rr - tt * G) * c.D + d, y);
    }
  }
}

// Joins the slices of the sequences that were cut: a workgroup to a (sequence, tile, head) item, found as above among the first slices.
template <int DP, int OUT>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttn a, PagedCache c, PagedBatch b, PagedPlan p, const float* ws) {
  const PagedItem it = paged_item(b, c.page_shift, c.heads, PA_ROWS, p, blockIdx.x);
  if (!it.found || it.split != 0 || it.splits == 1 || it.first + (long long)(it.splits - 1) * it.step >= p.slots) return;
  const int G = p.group, live_rows = it.s.T * G;
  const float* offs = ws + (long long)p.slots * PA_ROWS * DP;
  const float* den = offs + (long long)p.slots * PA_ROWS;
  for (int e = threadIdx.x; e < PA_ROWS * (DP / 4); e += 256) {
    const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
    const int rr = it.tile * PA_ROWS + r;
    if (rr >= live_rows || d >= c.D) continue;
    float least = PA_EMPTY;
    for (int s = 0; s < it.splits; ++s) {
      const float o = offs[(it.first + (long long)s * it.step) * PA_ROWS + r];
      least = o < least ? o : least;
    }
    float y[4] = {0, 0, 0, 0}, l = 0;
    for (int s = 0; s < it.splits; ++s) {
      const long long slot = it.first + (long long)s * it.step;
      const float scale = __builtin_amdgcn_exp2f(least - offs[slot * PA_ROWS + r]);
      const v4f v = *reinterpret_cast<const v4f*>(ws + (slot * PA_ROWS + r) * DP + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i] * scale;
      l += den[slot * PA_ROWS + r] * scale;
    }
    const float f = l > 0.0f ? a.alpha_pv * 1024.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = l > 0.0f ? y[i] * f : 0.0f;
    const int tt = rr / G;
    store4<OUT>(a.out, ((long long)(it.s.row0 + tt) * a.q_heads + it.head * G + rr - tt * G) * c.D + d, y);
  }
}

// Items that a batch can make: one to each (sequence, key head, 16 rows), and the slices beyond that.
static long long paged_units(long long rows, long long seqs, long long group, long long kv_heads, int tile) {
  return kv_heads * (seqs + rows * group / tile);
}
static bool paged_cuts(long long capacity) { return capacity > PA_MIN_SLICE; }
static long long paged_slots(long long rows, long long seqs, long long group, long long kv_heads) {
  return paged_units(rows, seqs, group, kv_heads, PA_ROWS) + PA_TARGET + 8;
}
static int paged_dp(long long D) { return D <= 64 ? 64 : 128; }

long long paged_attn_workspace_bytes(long long rows, long long seqs, long long q_heads, long long kv_heads, long long D,
                                     long long capacity) {
  if (rows <= 0 || seqs <= 0 || kv_heads <= 0 || !paged_cuts(capacity)) return 0;
  return paged_slots(rows, seqs, q_heads / kv_heads, kv_heads) * PA_ROWS * (paged_dp(D) + 2) * 4;
}

template <int DP, int OUT>
static void launch_rows(const PagedAttn& a, const PagedCache& c, const PagedBatch& b, const PagedPlan& p, float* ws, unsigned grid,
                        hipStream_t stream) {
  hipLaunchKernelGGL((paged_attn_rows_kernel<DP, OUT>), dim3(grid), dim3(PA_WAVES * 64), 0, stream, a, c, b, p, ws);
  if (p.target != 0)
    hipLaunchKernelGGL((paged_attn_join_kernel<DP, OUT>), dim3(grid), dim3(256), 0, stream, a, c, b, p, ws);
}

int launch_paged_attn_s8(int out_type, const PagedAttn& a, const PagedCache& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream) {
  if (b.rows == 0 || a.q_heads == 0) return TI_OK;
  PagedPlan p;
  p.group = a.q_heads / c.heads;
  const long long capacity = (long long)b.per_seq << c.page_shift;
  const long long need = paged_attn_workspace_bytes(b.rows, b.seqs, a.q_heads, c.heads, c.D, capacity);
  const bool cut = need > 0 && workspace != nullptr && workspace_bytes >= need;
  p.target = cut ? PA_TARGET : 0;
  p.slots = cut ? (int)paged_slots(b.rows, b.seqs, p.group, c.heads) : 0;
  const long long grid = cut ? p.slots : paged_units(b.rows, b.seqs, p.group, c.heads, PA_ROWS);
  if (grid > 0x7fffff) return fail(TI_ERR_INVALID_ARG, "paged_attn_s8: %lld work items", grid);
  float* ws = static_cast<float*>(workspace);
  const unsigned g = grid > 0 ? (unsigned)grid : 1u;
  if (paged_dp(c.D) == 64) {
    if (out_type == PT_S8) launch_rows<64, PT_S8>(a, c, b, p, ws, g, stream);
    else if (out_type == PT_F16) launch_rows<64, PT_F16>(a, c, b, p, ws, g, stream);
    else launch_rows<64, PT_BF16>(a, c, b, p, ws, g, stream);
  } else {
    if (out_type == PT_S8) launch_rows<128, PT_S8>(a, c, b, p, ws, g, stream);
    else if (out_type == PT_F16) launch_rows<128, PT_F16>(a, c, b, p, ws, g, stream);
    else launch_rows<128, PT_BF16>(a, c, b, p, ws, g, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_attn_s8 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

}  // namespace ti
