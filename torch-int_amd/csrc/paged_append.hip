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

// s8 of a whole number in fp32 (the conversion saturates, and makes 0 of NaN)
__device__ __forceinline__ int s8_of_whole(float n) {
  int i;
  asm("v_cvt_i32_f32 %0, %1" : "=v"(i) : "v"(n));
  return i < -128 ? -128 : i > 127 ? 127 : i;
}

// s8(rint(x alpha)) with the product unrounded.  A border between two results is an fp32 number, and rounding to fp32 passes
// none, so y = fl(x alpha) decides unless it is a border itself: then the remainder, which one FMA gives exactly, does.
__device__ __forceinline__ int s8_of_product(float x, float alpha) {
  const float y = x * alpha, n = __builtin_rintf(y), rest = __builtin_fmaf(x, alpha, -y);
  const bool border = __builtin_fabsf(y - n) == 0.5f && rest != 0.0f;
  return s8_of_whole(border ? y + __builtin_copysignf(0.5f, rest) : n);
}

// s8(rint((p c + q s) alpha)) in fp32.  Three roundings and one of the bound's own are off by less than 2^-22 (|p c| + |q s|) alpha
// together, the fp64 chain by 2^-51 of it; `far` keeps the bits of the largest |y - rint y| + twice that.  A result whose figure
// stays below one half is the fp64 chain's; infinities and NaN have larger bits than any number.
__device__ __forceinline__ int s8_of_turned(float p, float c, float q, float s, float alpha, float bound, unsigned& far) {
  const float t = q * s, r = __builtin_fmaf(p, c, t), w = __builtin_fmaf(__builtin_fabsf(p), __builtin_fabsf(c), __builtin_fabsf(t));
  const float y = r * alpha, n = __builtin_rintf(y);
  const unsigned bits = __float_as_uint(__builtin_fabsf(__builtin_fmaf(w, bound, __builtin_fabsf(y - n))));
  far = far > bits ? far : bits;
  return s8_of_whole(n);
}

__device__ __forceinline__ int2 pack8(const int (&o)[8]) {
  int2 r;
  r.x = (o[0] & 255) | (o[1] & 255) << 8 | (o[2] & 255) << 16 | o[3] << 24;
  r.y = (o[4] & 255) | (o[5] & 255) << 8 | (o[6] & 255) << 16 | o[7] << 24;
  return r;
}

// One row to blockIdx.x; the threads of a block are the 16-element pieces of some heads, the keys', then the values', then the
// queries'.  A piece is 16 neighbouring elements, or where pairs lie half apart 8 elements and their 8 partners.
// Memory and vector ALUs are about level: 8192 rows of 32 + 2 x 8 heads of 128 fp16, 155 MB, take 37 us (4.2 TB/s; in fp64 alone 44),
// 28 of them 350 instructions a wave, of which 130 look up rows and addresses; 2036 rows of 3 x 32 heads fp32, 125 MB, 27 us (4.6).
// Several rows to a block, the next row's elements ahead of the present one's, needs 98 registers instead of 66 and took 36 us for the
// second.
template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend a, PagedCache c, PagedBatch b, int pieces, int per_block) {
  const int row = blockIdx.x;
  const int unit = (int)(threadIdx.x * (65536u / (unsigned)pieces + 1u) >> 16);  // threadIdx.x / pieces, for 256 by up to 8
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
  const T* src = which == 0   ? static_cast<const T*>(a.key) + row * a.k_row + h * a.k_head
                 : which == 1 ? static_cast<const T*>(a.value) + row * a.v_row + h * a.v_head
                              : static_cast<const T*>(a.query) + row * a.q_row + h * a.q_head;
  Raw8<T> x0, x1;  // on their way while the row's place is looked up
  x0.load(src + d0);
  x1.load(src + d1);
  // the row's sequence: how many of them end at or before it (all lanes of the wave take part)
  int seq = 0;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63);
    const unsigned long long ended = __ballot(i < b.seqs && b.cu[i < b.seqs ? i + 1 : b.seqs] <= row);
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
    if (mine) position = s.len - s.T + (row - s.row0);
  }
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
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, a, c, b, pieces, per_block); };
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
