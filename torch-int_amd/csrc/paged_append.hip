// Appending keys and values to a paged int8 cache (and quantising the queries beside them): for every new row, its sequence
// from cu_new, its position from the sequence's length, its slot from the block table; then
//   y = x, or for a rotated pair (x1, x2) with (c, s) of the position: y1 = x1 c - x2 s, y2 = x2 c + x1 s
//   cache = s8(rint(clamp(alpha * y))),  NaN -> 0.
// The bytes are those of a plain fp64 chain of the formula (products of two fp32 values are exact there, so they depend on no
// order of operations), but the work is fp32, at twice the rate and without conversions: a result that lies too near a border
// between two bytes to be told from fp32 is done again in fp64 (of normal keys at scales of 1/32 about one piece in 500).
#include <hip/hip_fp16.h>
#include "paged.h"

namespace ti {

template <typename T>
__device__ __forceinline__ float as_float(T x) { return (float)x; }
struct bf16_bits { unsigned short u; };
template <>
__device__ __forceinline__ float as_float<bf16_bits>(bf16_bits x) { return __uint_as_float((unsigned)x.u << 16); }

// Eight neighbouring elements as they lie in memory, and their values.
template <typename T>
struct Raw8 {
  T x[8];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<v4i*>(x)[0] = reinterpret_cast<const v4i*>(p)[0];
      reinterpret_cast<v4i*>(x)[1] = reinterpret_cast<const v4i*>(p)[1];
    } else if constexpr (sizeof(T) == 2) {
      reinterpret_cast<v4i*>(x)[0] = reinterpret_cast<const v4i*>(p)[0];
    } else {
      reinterpret_cast<int2*>(x)[0] = reinterpret_cast<const int2*>(p)[0];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return as_float(x[i]); }
};

// s8 of a value in fp64: NaN becomes 0
__device__ __forceinline__ int s8_of(double y) {
  y = __builtin_rint(y);
  y = y < -128.0 ? -128.0 : y > 127.0 ? 127.0 : y;
  return y == y ? (int)y : 0;
}

// 1.5 * 2^23: a number added to it in one FMA is rounded, half to even, to a whole one, which the low bits then are.
constexpr float WHOLE = 12582912.0f;
// the low byte of what this returns is the s8 of n - WHOLE, for any n but NaN
__device__ __forceinline__ int byte_of(float n) { return __float_as_int(__builtin_amdgcn_fmed3f(n, WHOLE - 128.0f, WHOLE + 127.0f)); }

// s8(rint(x alpha)) in the low byte, the product unrounded; NaN becomes 0
__device__ __forceinline__ int s8_of_product(float x, float alpha) {
  const float n = __builtin_fmaf(x, alpha, WHOLE);
  return n == n ? byte_of(n) : 0;
}

// s8(rint((p c + q s) alpha)) in the low byte, in fp32.  The two roundings, and the bound's own, are off by less than
// 2^-22 (|p c| + |q s|) alpha together, the fp64 chain by 2^-51 of it; `far` keeps the bits of the largest |y - rint y| + twice
// that.  A result whose figure stays below one half is the fp64 chain's; infinities and NaN have larger bits than any number, and
// figures of numbers too large for WHOLE are above one half as well.
__device__ __forceinline__ int s8_of_turned(float p, float c, float q, float s, float alpha, float bound, unsigned& far) {
  const float t = q * s, r = __builtin_fmaf(p, c, t), w = __builtin_fmaf(__builtin_fabsf(p), __builtin_fabsf(c), __builtin_fabsf(t));
  const float n = __builtin_fmaf(r, alpha, WHOLE), d = __builtin_fmaf(r, alpha, -(n - WHOLE));
  const unsigned bits = __float_as_uint(__builtin_fabsf(__builtin_fmaf(w, bound, __builtin_fabsf(d))));
  far = far > bits ? far : bits;
  return byte_of(n);
}

// the low bytes of eight
__device__ __forceinline__ int2 pack8(const int (&o)[8]) {
  auto four = [](int x, int y, int z, int w) {
    return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400), __builtin_amdgcn_perm(y, x, 0x0c0c0400), 0x05040100);
  };
  return make_int2(four(o[0], o[1], o[2], o[3]), four(o[4], o[5], o[6], o[7]));
}

// One row to blockIdx.x; the threads of a block are the 16-element pieces of some heads, the keys', then the values', then the
// queries'.  A piece is 16 neighbouring elements, or where pairs lie half apart 8 elements and their 8 partners.
// At the rate of a copy: 8192 rows of 32 + 2 x 8 heads of 128 fp16, 155 MB, take 29.4 us (5.3 TB/s), 2036 rows of 3 x 32 heads fp32,
// 125 MB, 23.9 us (5.2).  That needs few instructions (280 a wave; in fp64 they took 44 us of the first) and the row's
// elements on their way before its place is known, behind the one load that begins the search (33.9 us in front of it).  Several rows
// to a block, the next row's elements ahead of the present one's, needs 98 registers instead of 66 and made the second 36 us.
template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend a, PagedCache c, PagedBatch b, int pieces, int per_piece,
                                                            int per_block) {
  const int row = blockIdx.x;
  const int unit = (int)(threadIdx.x * (unsigned)per_piece >> 16);  // threadIdx.x / pieces
  const int piece = threadIdx.x - unit * pieces;
  const int head = blockIdx.y * per_block + unit;
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  const bool real = unit < per_block && head < heads;
  const int which = !real || head < c.heads ? 0 : head < 2 * c.heads ? 1 : 2;  // key, value, query
  const int h = real ? head - (which == 0 ? 0 : which * c.heads) : 0;
  const int rot = a.cos_sin != nullptr && which != 1 ? a.rot : 0;
  const bool turned = piece * 16 < rot;
  const bool apart = turned && !a.neighbours;
  const int d0 = apart ? piece * 8 : piece * 16, d1 = apart ? rot / 2 + piece * 8 : piece * 16 + 8;
  // the row's sequence: how many of them end at or before it (all lanes of the wave take part); the first 64 ends are asked for in
  // front of the row's elements, which are on their way while its place is looked up
  const int lane = threadIdx.x & 63;
  int end = b.cu[lane < b.seqs ? lane + 1 : b.seqs];
  const T* const key = static_cast<const T*>(a.key) + row * a.k_row;
  const T* const value = static_cast<const T*>(a.value) + row * a.v_row;
  const T* const query = static_cast<const T*>(a.query) + row * a.q_row;
  const T* src = (which == 0 ? key : which == 1 ? value : query) + h * (which == 0 ? a.k_head : which == 1 ? a.v_head : a.q_head);
  Raw8<T> x0, x1;
  x0.load(src + d0);
  x1.load(src + d1);
  int seq = 0;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    const int i = i0 + lane;
    if (i0 > 0) end = b.cu[i < b.seqs ? i + 1 : b.seqs];
    const unsigned long long ended = __ballot(i < b.seqs && end <= row);
    seq += __popcll(ended);
    if (ended != ~0ull) break;
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  if (!real) return;
  int position = -1;
  bool mine = false;
  if (seq < b.seqs) {
    const PagedSeq s = paged_seq(b, c.page_shift, seq);
    mine = row >= s.row0 && row < s.row0 + s.T;
    if (mine) position = s.end - s.T + (row - s.row0);
    if (position >= s.len) position = -1;  // no page for it
  }
  const bool live = position >= 0 && (a.cos_sin == nullptr || position < a.positions);
  int8_t* dst = nullptr;
  if (which == 2) {
    dst = a.q_out + ((long long)row * a.q_heads + h) * c.D;
    if (!live) {  // a row of no sequence, or one whose position is before the first, beyond the pages or beyond the angles
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
  const float alpha = which == 0 ? a.alpha_k : which == 1 ? a.alpha_v : a.alpha_q;
  int o0[8], o1[8];
  if (!turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o0[i] = s8_of_product(x0[i], alpha);
      o1[i] = s8_of_product(x1[i], alpha);
    }
  } else {
    Raw8<float> cs, sn;
    const float* at = a.cos_sin + (long long)position * a.rot + piece * 8;
    cs.load(at);
    sn.load(at + a.rot / 2);
    float p[8], q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float here = x0[i], there = x1[i], even = i < 4 ? x0[2 * i % 8] : x1[2 * i % 8], odd = i < 4 ? x0[2 * i % 8 + 1] : x1[2 * i % 8 + 1];
      p[i] = apart ? here : even;
      q[i] = apart ? there : odd;
    }
    unsigned far = 0;
    const float bound = __builtin_fabsf(alpha) * 0x1p-21f + 0x1p-126f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o0[i] = s8_of_turned(p[i], cs[i], q[i], -sn[i], alpha, bound, far);
      o1[i] = s8_of_turned(q[i], cs[i], p[i], sn[i], alpha, bound, far);
    }
    if (far >= __float_as_uint(0.5f)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double u = p[i], w = q[i], co = cs[i], si = sn[i];
        o0[i] = s8_of((u * co - w * si) * alpha);
        o1[i] = s8_of((w * co + u * si) * alpha);
      }
    }
  }
  int2 first = pack8(o0), second = pack8(o1);
  if (turned && !apart) {  // the pairs' firsts and seconds, byte by byte in turn
    const int2 u = first, w = second;
    first = make_int2(__builtin_amdgcn_perm(w.x, u.x, 0x05010400), __builtin_amdgcn_perm(w.x, u.x, 0x07030602));
    second = make_int2(__builtin_amdgcn_perm(w.y, u.y, 0x05010400), __builtin_amdgcn_perm(w.y, u.y, 0x07030602));
  }
  *reinterpret_cast<int2*>(dst + d0) = first;
  *reinterpret_cast<int2*>(dst + d1) = second;
}

int launch_paged_kv_append_s8(int type, const PagedAppend& a, const PagedCache& c, const PagedBatch& b, hipStream_t stream) {
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  if (b.rows == 0 || heads == 0) return TI_OK;
  const int pieces = c.D / 16;
  // as few blocks to a row as 256 threads allow, and as even
  const int blocks = (heads * pieces + 255) / 256;
  const int most = 256 / pieces, even = (heads + blocks - 1) / blocks, per_block = even < most ? even : most;
  const int threads = (per_block * pieces + 63) & ~63;
  const dim3 grid((unsigned)b.rows, (unsigned)((heads + per_block - 1) / per_block));
  auto launch = [&](auto kernel) {  // (65536 / pieces + 1 is exact for 256 threads by up to 8 pieces)
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, a, c, b, pieces, 65536 / pieces + 1, per_block);
  };
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
