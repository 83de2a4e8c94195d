// Appending keys and values to a paged int8 cache (and quantising the queries beside them): for every new row, its sequence
// from cu_new, its position from the sequence's length, its slot from the block table; then
//   y = x, or for a rotated pair (x1, x2) with (c, s) of the position: y1 = x1 c - x2 s, y2 = x2 c + x1 s
//   cache = s8(rint(clamp(alpha * y))),  NaN -> 0.
// The rounding is that of fp64 arithmetic: products of two fp32 values are exact there, so the bits do not depend on an order
// of fp32 operations and a plain fp64 chain of the same formula gives the same bytes.
#include <hip/hip_fp16.h>
#include "paged.h"

namespace ti {

template <typename T>
__device__ __forceinline__ float as_float(T x) { return (float)x; }
struct bf16_bits { unsigned short u; };
template <>
__device__ __forceinline__ float as_float<bf16_bits>(bf16_bits x) { return __uint_as_float((unsigned)x.u << 16); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  T raw[8];
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<v4i*>(raw)[0] = reinterpret_cast<const v4i*>(p)[0];
    reinterpret_cast<v4i*>(raw)[1] = reinterpret_cast<const v4i*>(p)[1];
  } else if constexpr (sizeof(T) == 2) {
    reinterpret_cast<v4i*>(raw)[0] = reinterpret_cast<const v4i*>(p)[0];
  } else {
    reinterpret_cast<int2*>(raw)[0] = reinterpret_cast<const int2*>(p)[0];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = as_float(raw[i]);
}

// s8 of a value in fp64: NaN becomes 0
__device__ __forceinline__ int s8_of(double y) {
  y = __builtin_rint(y);
  y = y < -128.0 ? -128.0 : y > 127.0 ? 127.0 : y;
  return y == y ? (int)y : 0;
}

__device__ __forceinline__ int2 pack8(const int (&o)[8]) {
  int2 r;
  r.x = (o[0] & 255) | (o[1] & 255) << 8 | (o[2] & 255) << 16 | o[3] << 24;
  r.y = (o[4] & 255) | (o[5] & 255) << 8 | (o[6] & 255) << 16 | o[7] << 24;
  return r;
}

// One row to blockIdx.x; the threads of a block are the 16-element pieces of some heads, the keys', then the values', then the
// queries'.  A piece is 16 neighbouring elements, or where pairs lie half apart 8 elements and their 8 partners.
template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend a, PagedCache c, PagedBatch b, int pieces, int per_block) {
  const int row = blockIdx.x;
  // the row's sequence: how many of them end at or before it (all lanes of the wave take part)
  int seq = 0;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63);
    const unsigned long long ended = __ballot(i < b.seqs && b.cu[i < b.seqs ? i + 1 : b.seqs] <= row);
    seq += __popcll(ended);
    if (ended != ~0ull) break;
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  const int unit = (int)(threadIdx.x * (65536u / (unsigned)pieces + 1u) >> 16);  // threadIdx.x / pieces, for 256 by up to 8
  const int piece = threadIdx.x - unit * pieces;
  const int head = blockIdx.y * per_block + unit;
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  if (unit >= per_block || head >= heads) return;
  const int which = head < c.heads ? 0 : head < 2 * c.heads ? 1 : 2;  // key, value, query
  const int h = head - (which == 0 ? 0 : which * c.heads);
  int position = -1;
  bool mine = false;
  if (seq < b.seqs) {
    const PagedSeq s = paged_seq(b, c.page_shift, seq);
    mine = row >= s.row0 && row < s.row0 + s.T;
    if (mine) position = s.len - s.T + (row - s.row0);
  }
  const int rot = a.cos_sin != nullptr && which != 1 ? a.rot : 0;
  const bool turned = piece * 16 < rot;
  const bool apart = turned && !a.neighbours;
  const int d0 = apart ? piece * 8 : piece * 16, d1 = apart ? rot / 2 + piece * 8 : piece * 16 + 8;
  const bool live = position >= 0 && (a.cos_sin == nullptr || position < a.positions);
  int8_t* dst = nullptr;
  if (which == 2) {
    dst = a.q_out + ((long long)row * a.q_heads + h) * c.D;
    if (!live) {  // a row of no sequence, or one whose position is before the first or beyond the table
      if (a.fill || mine) {
        *reinterpret_cast<int2*>(dst + d0) = make_int2(0, 0);
        *reinterpret_cast<int2*>(dst + d1) = make_int2(0, 0);
      }
      return;
    }
  } else {
    if (!live) return;
    const int page = b.table[(long long)seq * b.per_seq + (position >> c.page_shift)];
    if (page < 0 || page >= c.pages) return;
    const int off = position & ((1 << c.page_shift) - 1);
    dst = which == 0 ? c.k + (long long)page * c.k_page + h * c.k_head + (long long)off * c.k_token
                     : c.v + (long long)page * c.v_page + h * c.v_head + (long long)off * c.v_token;
  }
  const T* src = which == 0   ? static_cast<const T*>(a.key) + row * a.k_row + h * a.k_head
                 : which == 1 ? static_cast<const T*>(a.value) + row * a.v_row + h * a.v_head
                              : static_cast<const T*>(a.query) + row * a.q_row + h * a.q_head;
  const double alpha = which == 0 ? a.alpha_k : which == 1 ? a.alpha_v : a.alpha_q;
  float x0[8], x1[8];
  load8(src + d0, x0);
  load8(src + d1, x1);
  int o0[8], o1[8];
  if (!turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o0[i] = s8_of((double)x0[i] * alpha);
      o1[i] = s8_of((double)x1[i] * alpha);
    }
  } else {
    float cs[8], sn[8];
    const float* at = a.cos_sin + (long long)position * a.rot + piece * 8;
    load8(at, cs);
    load8(at + a.rot / 2, sn);
    if (apart) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double p = x0[i], q = x1[i], co = cs[i], si = sn[i];
        o0[i] = s8_of((p * co - q * si) * alpha);
        o1[i] = s8_of((q * co + p * si) * alpha);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double p = i < 4 ? x0[2 * i % 8] : x1[2 * i % 8], q = i < 4 ? x0[2 * i % 8 + 1] : x1[2 * i % 8 + 1];
        const double co = cs[i], si = sn[i];
        const int u = s8_of((p * co - q * si) * alpha), w = s8_of((q * co + p * si) * alpha);
        if (i < 4) {
          o0[2 * i % 8] = u;
          o0[2 * i % 8 + 1] = w;
        } else {
          o1[2 * i % 8] = u;
          o1[2 * i % 8 + 1] = w;
        }
      }
    }
  }
  *reinterpret_cast<int2*>(dst + d0) = pack8(o0);
  *reinterpret_cast<int2*>(dst + d1) = pack8(o1);
}

int launch_paged_kv_append_s8(int type, const PagedAppend& a, const PagedCache& c, const PagedBatch& b, hipStream_t stream) {
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  if (b.rows == 0 || heads == 0) return TI_OK;
  const int pieces = c.D / 16;
  int per_block = 256 / pieces;
  if (per_block > heads) per_block = heads;
  const dim3 grid((unsigned)b.rows, (unsigned)((heads + per_block - 1) / per_block));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a, c, b, pieces, per_block); };
  switch (type) {
    case PT_F32: launch(paged_append_kernel<float>); break;
    case PT_F16: launch(paged_append_kernel<_Float16>); break;
    case PT_BF16: launch(paged_append_kernel<bf16_bits>); break;
    default: launch(paged_append_kernel<int8_t>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_kv_append_s8 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

}  // namespace ti
