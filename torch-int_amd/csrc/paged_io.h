// What the kernels that write rows to pages, or read them back, share: rows' elements, their rounding, and where a row belongs.
#pragma once
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

// the low bytes of eight
__device__ __forceinline__ int2 pack8(const int (&o)[8]) {
  auto four = [](int x, int y, int z, int w) {
    return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400), __builtin_amdgcn_perm(y, x, 0x0c0c0400), 0x05040100);
  };
  return make_int2(four(o[0], o[1], o[2], o[3]), four(o[4], o[5], o[6], o[7]));
}

// How many sequences end at or before `row`: the number of the sequence that it can belong to.  All lanes of the wave take part.
// `end` is what lane i has of the first 64 ends, asked for by paged_ends.
__device__ __forceinline__ int paged_ends(const PagedBatch& b) {
  const int lane = threadIdx.x & 63;
  return b.cu[lane < b.seqs ? lane + 1 : b.seqs];
}
__device__ __forceinline__ int paged_seq_of(const PagedBatch& b, int row, int end) {
  const int lane = threadIdx.x & 63;
  int seq = 0;
  for (int i0 = 0; i0 < b.seqs; i0 += 64) {
    const int i = i0 + lane;
    if (i0 > 0) end = b.cu[i < b.seqs ? i + 1 : b.seqs];
    const unsigned long long ended = __ballot(i < b.seqs && end <= row);
    seq += __popcll(ended);
    if (ended != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(seq);
}

// A new row's sequence and position; -1 where it has none, or no page in the table.
struct PagedPlace {
  int seq, position;
  bool mine;  // it belongs to a sequence
};
__device__ __forceinline__ PagedPlace paged_place(const PagedBatch& b, int page_shift, int row, int seq) {
  PagedPlace p = {seq, -1, false};
  if (seq < b.seqs) {
    const PagedSeq s = paged_seq(b, page_shift, seq);
    p.mine = row >= s.row0 && row < s.row0 + s.T;
    if (p.mine) p.position = s.end - s.T + (row - s.row0);
    if (p.position >= s.len) p.position = -1;
  }
  return p;
}

// The same with fewer trips to memory: lane i of a wave asks for the end and the length of sequence i at once, so that of the first 64
// sequences nothing has to be asked for when it is known which one a row belongs to.
struct PagedAsked {
  int first, end, len;
};
__device__ __forceinline__ PagedAsked paged_ask(const PagedBatch& b) {
  const int lane = threadIdx.x & 63;
  return PagedAsked{b.cu[0], b.cu[lane < b.seqs ? lane + 1 : b.seqs], lane < b.seqs ? b.lens[lane] : 0};
}
__device__ __forceinline__ PagedPlace paged_place(const PagedBatch& b, int page_shift, int row, const PagedAsked& asked) {
  const int seq = paged_seq_of(b, row, asked.end);
  PagedPlace p = {seq, -1, false};
  if (seq < b.seqs) {
    PagedSeq s;
    if (seq < 64) {
      s = paged_seq(b, page_shift, seq == 0 ? asked.first : __builtin_amdgcn_readlane(asked.end, seq - 1),
                    __builtin_amdgcn_readlane(asked.end, seq), __builtin_amdgcn_readlane(asked.len, seq));
    } else {
      s = paged_seq(b, page_shift, seq);
    }
    p.mine = row >= s.row0 && row < s.row0 + s.T;
    if (p.mine) p.position = s.end - s.T + (row - s.row0);
    if (p.position >= s.len) p.position = -1;
  }
  return p;
}

}  // namespace ti
