// Writing keys and values to a paged cache in 4 bits, and reading them back.  For every new row, its sequence, position and page
// as in the int8 cache; then for each head
//   y = fp32(alpha x), or for a rotated pair (x1, x2) with (c, s) of the position fp32(alpha (x1 c - x2 s)), fp32(alpha (x2 c + x1 s))
// (in fp64, where products of two fp32 values are exact; NaN -> 0, cut off at +-57344), and for each group of a head's values
//   a = min(0, y), b = max(0, y),  step = the smallest number of its format with 15 step >= b - a,
//   z = rint(-a / step),  u = clamp(rint(y / step) + z, 0, 15):
// 0 is one of the 16 values, and none of the group's is further from its own than half a step.  A group of zeros has step 0.
//
// Quotients are rounded half to even exactly: y / step, 15 at most, is a product with 1 / step in fp64, off by less than 2^-38, and a
// quotient of a 24-bit number by a 7-bit one that is no tie is further than 2^-25 from any tie; so the multiply-add to 1.5 2^17,
// which rounds to multiples of 2^-35, makes ties exact ties, and adding 1.5 2^52 - 1.5 2^17 leaves the integer in the low word.
#include "paged_io.h"

namespace ti {

constexpr double S4_GRID = 196608.0, S4_INT = 6755399441055744.0 - 196608.0;  // 1.5 2^17, 1.5 2^52 less that

// The largest of the L lanes (4 or 8, neighbours) that share a head, in all of them.
template <int L>
__device__ __forceinline__ float lanes_max(float x) {
  auto step = [&](auto ctrl) {
    return __builtin_fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  x = step(std::integral_constant<int, 0xb1>());               // quad_perm: 1 0 3 2
  x = step(std::integral_constant<int, 0x4e>());               // quad_perm: 2 3 0 1
  if (L == 8) x = step(std::integral_constant<int, 0x141>());  // row_half_mirror
  return x;
}

// A group's word and how its values become codes.
struct S4Group {
  int word, zero;
  double inv;
  // low <= 0 <= high
  __device__ __forceinline__ S4Group(float low, float high) {
    const double span = (double)high - (double)low;
    // a step of the format at or below span / 15, then at most two up
    const float most = (float)span * (0.066666667f * (1.0f - 0x1p-20f));
    int h = __builtin_bit_cast(int, __builtin_amdgcn_cvt_pkrtz(most, 0.0f)) & S4_STEP;
    auto value = [](int h) { return (float)__builtin_bit_cast(_Float16, (unsigned short)h); };
#pragma unroll
    for (int i = 0; i < 2; ++i) h += (double)(15.0f * value(h)) < span ? 16 : 0;
    // 1 / step: the hardware's, off by 2^-22, and one step of Newton's, off by less than 2^-43
    const float s = value(h), r = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;
    inv = __builtin_fma(__builtin_fma(-(double)s, (double)r, 1.0), (double)r, (double)r);
    zero = whole(-low);
    word = h | zero;
  }
  __device__ __forceinline__ int whole(float y) const {
    const double n = __builtin_fma((double)y, inv, S4_GRID) + S4_INT;
    return (int)(unsigned)__builtin_bit_cast(unsigned long long, n);
  }
  __device__ __forceinline__ int code(float y) const {
    const int u = whole(y) + zero;
    return u < 0 ? 0 : u > 15 ? 15 : u;
  }
};

// s8(rint(v)) of a value in fp64 in the low byte, without a branch; NaN becomes 0
__device__ __forceinline__ int byte_of_double(double v) {
  const double n = __builtin_fmin(__builtin_fmax(v, -128.0), 127.0) + 6755399441055744.0;
  const int k = (int)(unsigned)__builtin_bit_cast(unsigned long long, n);
  return v == v ? k : 0;
}

// Rows of 16-bit queries, eight at a time
template <typename H>
__device__ __forceinline__ void store8h(void* to, const float (&y)[8]) {
  H h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (H)y[i];
  v4i w;
  __builtin_memcpy(&w, h, 16);
  *reinterpret_cast<v4i*>(to) = w;
}

// The wave's row and the first of its heads: `waves` of them to a row.
struct S4Wave {
  int row, head;
  __device__ __forceinline__ S4Wave(int waves, int lanes) {
    const int id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    row = (int)((unsigned)id / (unsigned)waves);
    head = (id - row * waves) * (64 / lanes);
  }
};

// L lanes to a head (the keys', then the values', then the queries'), of which lane p < D / 16 has the columns 8 p .. 8 p + 7 and their
// counterparts D / 2 further on: the bytes 8 p .. 8 p + 7 of its codes.
// 7001 rows of 32 + 2 x 8 heads of 128 fp16, rotated, 126 MB: 31.7 us (4.0 TB/s; a copy of as much runs at 5.0).  The vector ALUs are busy for
// 21 of them (some 330 instructions a wave, fp64 at the rate of fp32); waves are short chains of three trips to memory, so as many
// as fit: 64 registers, eight waves to a SIMD, where 90 made it 36.
template <typename T, int L>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 8 : sizeof(T) == 4 ? 6 : 4) void paged_append_s4_kernel(PagedAppend4 a, PagedCache4 c, PagedBatch b, int waves) {
  const S4Wave mine(waves, L);
  const int row = mine.row;
  if (row >= b.rows) return;
  const int head = mine.head + (threadIdx.x & 63) / L, lane = threadIdx.x % L;
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  const bool real = head < heads && lane * 16 < c.D;
  const int which = head >= heads || head < c.heads ? 0 : head < 2 * c.heads ? 1 : 2;  // key, value, query
  const int h = head >= heads ? 0 : head - (which == 0 ? 0 : which * c.heads);
  const int at = real ? lane * 8 : 0, half = c.D / 2;
  const int rot = a.cos_sin != nullptr && which != 1 ? a.rot : 0;
  const PagedAsked asked = paged_ask(b);
  const T* const src = which == 0 ? static_cast<const T*>(a.key) + row * a.k_row + h * a.k_head
                     : which == 1 ? static_cast<const T*>(a.value) + row * a.v_row + h * a.v_head
                                  : static_cast<const T*>(a.query) + row * a.q_row + h * a.q_head;
  Raw8<T> x[2];
  x[0].load(src + at);
  x[1].load(src + half + at);
  const PagedPlace place = paged_place(b, c.page_shift, row, asked);
  const int position = place.position;
  const bool live = position >= 0 && (a.cos_sin == nullptr || position < a.positions);
  if (!live) {  // the same for all of the wave: a row of no sequence, or one whose position is before the first, beyond pages or angles
    if (which == 2 && real && (a.fill || place.mine)) {
      const long long to = ((long long)row * a.q_heads + h) * c.D;
      if (a.q_type == PT_S8) {
        int8_t* out = static_cast<int8_t*>(a.q_out) + to;
        *reinterpret_cast<int2*>(out + at) = make_int2(0, 0);
        *reinterpret_cast<int2*>(out + half + at) = make_int2(0, 0);
      } else {
        uint16_t* out = static_cast<uint16_t*>(a.q_out) + to;
        *reinterpret_cast<v4i*>(out + at) = v4i{0, 0, 0, 0};
        *reinterpret_cast<v4i*>(out + half + at) = v4i{0, 0, 0, 0};
      }
    }
    return;
  }
  const int page = b.table[(long long)place.seq * b.per_seq + (position >> c.page_shift)];
  const float alpha = which == 0 ? a.alpha_k : which == 1 ? a.alpha_v : a.alpha_q;
  // take(q, i, v): element i of half q, turned and times alpha
  const float* const turn = a.cos_sin + (long long)position * a.rot;
  auto turned = [&](auto take) {
    if (rot == c.D && !a.neighbours) {  // the usual rotation: a lane has both elements of its pairs
      Raw8<float> cs, sn;
      cs.load(turn + at);
      sn.load(turn + half + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double p = x[0][i], w = x[1][i], co = cs[i], si = sn[i];
        take(0, i, __builtin_fma(p, co, -(w * si)) * (double)alpha);
        take(1, i, __builtin_fma(w, co, p * si) * (double)alpha);
      }
      return;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int d = q * half + at;
      if (d >= rot) {
#pragma unroll
        for (int i = 0; i < 8; ++i) take(q, i, (double)x[q][i] * (double)alpha);
      } else if (a.neighbours) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double co = turn[d / 2 + i], si = turn[rot / 2 + d / 2 + i], p = x[q][2 * i], w = x[q][2 * i + 1];
          take(q, 2 * i, __builtin_fma(p, co, -(w * si)) * (double)alpha);
          take(q, 2 * i + 1, __builtin_fma(w, co, p * si) * (double)alpha);
        }
      } else {
        const bool first = d < rot / 2;
        const int j = first ? d : d - rot / 2;
        Raw8<T> other;
        other.load(src + (first ? d + rot / 2 : j));
        Raw8<float> cs, sn;
        cs.load(turn + j);
        sn.load(turn + rot / 2 + j);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double p = x[q][i], w = other[i], si = first ? -sn[i] : sn[i];
          take(q, i, __builtin_fma(p, (double)cs[i], w * si) * (double)alpha);
        }
      }
    }
  };
  if (which == 2) {
    if (!real) return;
    const long long to = ((long long)row * a.q_heads + h) * c.D + at;
    if (a.q_type == PT_S8) {
      int o[2][8];
      turned([&](int q, int i, double v) { o[q][i] = byte_of_double(v); });
#pragma unroll
      for (int q = 0; q < 2; ++q) *reinterpret_cast<int2*>(static_cast<int8_t*>(a.q_out) + to + q * half) = pack8(o[q]);
    } else {
      float y[2][8];
      turned([&](int q, int i, double v) { y[q][i] = (float)v; });
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (a.q_type == PT_F16) store8h<_Float16>(static_cast<_Float16*>(a.q_out) + to + q * half, y[q]);
        else store8h<__bf16>(static_cast<__bf16*>(a.q_out) + to + q * half, y[q]);
      }
    }
    return;
  }
  float y[2][8];
  if (rot == 0) {  // one rounding, as that of the product in fp64
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[q][i] = x[q][i] * alpha;
  } else {
    turned([&](int q, int i, double v) { y[q][i] = (float)v; });
  }
  // the least and the largest, 0 among them; the instructions pass NaN over, which is looked for beside them
  float low[2], high[2];
  auto span = [&] {
    bool odd = false;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      low[q] = high[q] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        low[q] = __builtin_fminf(__builtin_fminf(low[q], y[q][i]), y[q][i + 1]);
        high[q] = __builtin_fmaxf(__builtin_fmaxf(high[q], y[q][i]), y[q][i + 1]);
        odd |= __builtin_isunordered(y[q][i], y[q][i + 1]);
      }
      odd |= low[q] < -S4_MOST || high[q] > S4_MOST;
    }
    return odd;
  };
  if (__builtin_expect(span(), 0)) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[q][i] = y[q][i] == y[q][i] ? __builtin_amdgcn_fmed3f(y[q][i], -S4_MOST, S4_MOST) : 0.0f;
    span();
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {  // idle lanes have nothing to say
    low[q] = -lanes_max<L>(real ? -low[q] : 0.0f);
    high[q] = lanes_max<L>(real ? high[q] : 0.0f);
  }
  if (c.groups == 1) {
    low[0] = low[1] = __builtin_fminf(low[0], low[1]);
    high[0] = high[1] = __builtin_fmaxf(high[0], high[1]);
  }
  const S4Group first(low[0], high[0]), second(low[1], high[1]);
  if (!real || page < 0 || page >= c.pages) return;
  const int off = position & ((1 << c.page_shift) - 1);
  int w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = first.code(y[0][i]) | second.code(y[1][i]) << 4;
  uint8_t* const dst = (which == 0 ? c.k : c.v) + (long long)page * c.page + h * c.head + (long long)off * c.token;
  *reinterpret_cast<int2*>(dst + at) = pack8(w);
  if (lane == 0) {
    char* const scale = reinterpret_cast<char*>(which == 0 ? c.k_scale : c.v_scale) + (long long)page * c.scale_page + h * c.scale_head;
    if (c.groups == 1) reinterpret_cast<uint16_t*>(scale)[off] = (uint16_t)first.word;
    else reinterpret_cast<unsigned*>(scale)[off] = (unsigned)(first.word | second.word << 16);
  }
}

// The way back: alpha s (u - z) of the positions that `cu` asks for, of the keys and of the values of a head by the same L lanes, which
// find their place once then: 30018 rows of 8 heads of 128 to bf16, 156 MB, 33.7 us (4.6 TB/s), 41 with lanes of their own.
template <int TYPE, int L>
__global__ __launch_bounds__(256) void paged_read_s4_kernel(PagedRead4 a, PagedCache4 c, PagedBatch b, int waves) {
  const S4Wave mine(waves, L);
  const int row = mine.row;
  if (row >= b.rows) return;
  const int h = mine.head + (threadIdx.x & 63) / L, lane = threadIdx.x % L;
  const PagedPlace place = paged_place(b, c.page_shift, row, paged_ask(b));
  if (!place.mine && !a.fill) return;
  int page = -1;
  if (place.position >= 0) page = b.table[(long long)place.seq * b.per_seq + (place.position >> c.page_shift)];
  if (h >= c.heads || lane * 16 >= c.D) return;
  const int at = lane * 8, half = c.D / 2;
  const bool there = page >= 0 && page < c.pages;
  int2 codes[2] = {};
  unsigned words[2] = {};
  if (there) {
    const int off = place.position & ((1 << c.page_shift) - 1);
    const long long code = (long long)page * c.page + h * c.head + (long long)off * c.token + at;
    const long long word = (long long)page * c.scale_page + h * c.scale_head + (long long)off * (2 * c.groups);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      codes[i] = *reinterpret_cast<const int2*>((i ? c.v : c.k) + code);
      const char* const w = reinterpret_cast<const char*>(i ? c.v_scale : c.k_scale) + word;
      words[i] = c.groups == 1 ? *reinterpret_cast<const uint16_t*>(w) * 0x10001u : *reinterpret_cast<const unsigned*>(w);
    }
  }
  const long long to = ((long long)row * c.heads + h) * c.D + at;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float alpha = i ? a.alpha_v : a.alpha_k;
    void* const out = i ? a.value : a.key;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned w = words[i] >> (16 * q);
      const float s = (float)__builtin_bit_cast(_Float16, (unsigned short)(w & S4_STEP)), z = (float)(int)(w & 15u);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned u = (unsigned)(j < 4 ? codes[i].x : codes[i].y) >> (8 * (j & 3) + 4 * q) & 15u;
        y[j] = s * ((float)u - z);  // exact
      }
      if constexpr (TYPE == PT_S8) {
        int o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = s8_of_product(y[j], alpha);
        *reinterpret_cast<int2*>(static_cast<int8_t*>(out) + to + q * half) = pack8(o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= alpha;
        if constexpr (TYPE == PT_F32) {
          float* p = static_cast<float*>(out) + to + q * half;
          reinterpret_cast<v4f*>(p)[0] = v4f{y[0], y[1], y[2], y[3]};
          reinterpret_cast<v4f*>(p)[1] = v4f{y[4], y[5], y[6], y[7]};
        } else if constexpr (TYPE == PT_F16) {
          store8h<_Float16>(static_cast<_Float16*>(out) + to + q * half, y);
        } else {
          store8h<__bf16>(static_cast<__bf16*>(out) + to + q * half, y);
        }
      }
    }
  }
}

// Whole waves to a row, four waves to a block.
struct S4Grid {
  int waves;
  dim3 grid;
  S4Grid(int rows, int heads, int lanes) : waves((heads * lanes + 63) / 64), grid((unsigned)(((long long)rows * waves + 3) / 4)) {}
};

int launch_paged_kv_append_s4(int type, const PagedAppend4& a, const PagedCache4& c, const PagedBatch& b, hipStream_t stream) {
  const int heads = 2 * c.heads + (a.query != nullptr ? a.q_heads : 0);
  if (b.rows == 0 || heads == 0) return TI_OK;
  const int lanes = c.D <= 64 ? 4 : 8;
  const S4Grid g(b.rows, heads, lanes);
  auto launch = [&](auto four, auto eight) {
    if (lanes == 4) hipLaunchKernelGGL(four, g.grid, dim3(256), 0, stream, a, c, b, g.waves);
    else hipLaunchKernelGGL(eight, g.grid, dim3(256), 0, stream, a, c, b, g.waves);
  };
  switch (type) {
    case PT_F32: launch(paged_append_s4_kernel<float, 4>, paged_append_s4_kernel<float, 8>); break;
    case PT_F16: launch(paged_append_s4_kernel<_Float16, 4>, paged_append_s4_kernel<_Float16, 8>); break;
    case PT_BF16: launch(paged_append_s4_kernel<bf16_bits, 4>, paged_append_s4_kernel<bf16_bits, 8>); break;
    default: launch(paged_append_s4_kernel<int8_t, 4>, paged_append_s4_kernel<int8_t, 8>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_kv_append_s4 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

int launch_paged_kv_read_s4(int type, const PagedRead4& a, const PagedCache4& c, const PagedBatch& b, hipStream_t stream) {
  if (b.rows == 0) return TI_OK;
  const int lanes = c.D <= 64 ? 4 : 8;
  const S4Grid g(b.rows, c.heads, lanes);
  auto launch = [&](auto four, auto eight) {
    if (lanes == 4) hipLaunchKernelGGL(four, g.grid, dim3(256), 0, stream, a, c, b, g.waves);
    else hipLaunchKernelGGL(eight, g.grid, dim3(256), 0, stream, a, c, b, g.waves);
  };
  switch (type) {
    case PT_F32: launch(paged_read_s4_kernel<PT_F32, 4>, paged_read_s4_kernel<PT_F32, 8>); break;
    case PT_F16: launch(paged_read_s4_kernel<PT_F16, 4>, paged_read_s4_kernel<PT_F16, 8>); break;
    case PT_BF16: launch(paged_read_s4_kernel<PT_BF16, 4>, paged_read_s4_kernel<PT_BF16, 8>); break;
    default: launch(paged_read_s4_kernel<PT_S8, 4>, paged_read_s4_kernel<PT_S8, 8>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(TI_ERR_LAUNCH, "paged_kv_read_s4 launch: %s", hipGetErrorString(e));
  return TI_OK;
}

}  // namespace ti
