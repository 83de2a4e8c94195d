// What the kernels over a paged KV cache share: the cache, the batch, and how a workgroup finds its sequence.
#pragma once
#include "ti_common.h"

namespace ti {

struct PagedCache {
  int8_t* k;
  int8_t* v;
  long long k_page, k_head, v_page, v_head;  // bytes from page to page and from head to head
  int k_token, v_token;                      // bytes from position to position inside a page
  int pages, page_shift;                     // pages in the pool; log2 of the positions of a page (4 or more)
  int heads, D;                              // key/value heads, head size (a multiple of 16 up to 128)
};

struct PagedBatch {
  const int* table;  // [seqs, per_seq] pages of each sequence
  const int* lens;   // [seqs] cached positions, the new ones counted
  const int* cu;     // [seqs + 1] first new row of each sequence
  int per_seq, seqs, rows;
};

// One sequence of a batch.  The three arrays are device memory that the host never sees, so whatever they hold is brought
// into range here: no row, position or table entry outside the tensors is ever formed from row0, T and len.  `end` is the
// length before it is cut off (up to 2^30, which is beyond all the 2^28 positions that there can be pages for): appending keeps to
// it, since a new token that moved down with the cut would be written over a position that is somebody else's.
struct PagedSeq {
  int row0, T, len, end;  // first row, new tokens, cached positions that there are pages for, all positions
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int page_shift, int lo, int hi, int len) {
  PagedSeq s;
  const int cap = b.per_seq << page_shift;
  lo = lo < 0 ? 0 : lo > b.rows ? b.rows : lo;
  hi = hi < lo ? lo : hi > b.rows ? b.rows : hi;
  s.row0 = lo;
  s.T = hi - lo;
  s.end = len < 0 ? 0 : len < (1 << 30) ? len : 1 << 30;
  s.len = s.end > cap ? cap : s.end;
  return s;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int page_shift, int i) {
  return paged_seq(b, page_shift, b.cu[i], b.cu[i + 1], b.lens[i]);
}

enum PagedType : int { PT_F32 = 0, PT_F16 = 1, PT_BF16 = 2, PT_S8 = 3 };

// paged_append.hip
struct PagedAppend {
  const void *key, *value, *query;                        // query may be null
  long long k_row, k_head, v_row, v_head, q_row, q_head;  // elements
  int8_t* q_out;                                          // [rows, q_heads, D] packed
  int q_heads;
  const float* cos_sin;  // [positions, rot]: cosines, then sines; null: nothing is rotated
  int rot, positions;
  bool neighbours, fill;  // pairs are neighbours instead of half apart; rows of no sequence of q_out become zeros
  float alpha_q, alpha_k, alpha_v;
};
int launch_paged_kv_append_s8(int type, const PagedAppend& a, const PagedCache& c, const PagedBatch& b, hipStream_t stream);

// paged_attn.hip
struct PagedAttn {
  const int8_t* q;
  long long q_row, q_head;  // bytes
  int q_heads;
  void* out;  // [rows, q_heads, D] packed
  float alpha_qk, alpha_pv;
  bool fill;  // rows of no sequence become zeros
  int* arrivals;  // zeros, kept for the stream, or null
  long long arrivals_count;
};
long long paged_attn_arrivals(long long rows, long long seqs, long long q_heads, long long kv_heads, long long capacity);
long long paged_attn_workspace_bytes(long long rows, long long seqs, long long q_heads, long long kv_heads, long long D,
                                     long long capacity);
int launch_paged_attn_s8(int out_type, const PagedAttn& a, const PagedCache& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream);

// The same in 4 bits.  Byte j of a row of D / 2 holds the code u of column j in its low four bits and that of column D / 2 + j in
// the others.  A row has `groups` words, one for the whole head or one for each half (the low nibbles, the high ones): bits 4 to 14
// are those of an fp16 number, the step s, with 7 significant bits; bits 0 to 3 are z, and a value is s (u - z).  Seven bits
// times four are exact in fp16, so kernels that compute in fp16 compute with the very values.
struct PagedCache4 {
  uint8_t *k, *v;
  uint16_t *k_scale, *v_scale;               // [pages, heads, page, groups], the last two packed
  long long page, head, scale_page, scale_head;  // bytes from page to page and from head to head, of codes and of words
  int token;              // bytes from position to position inside a page
  int pages, page_shift;  // pages in the pool; log2 of the positions of a page (4 or more)
  int heads, D, groups;   // key/value heads, head size (a multiple of 16 from 32 to 128), words of a row (1 or 2)
};
constexpr int S4_STEP = 0x7ff0;        // a word's step
constexpr float S4_MOST = 57344.0f;    // values are cut off here: with half a step more they still are fp16 numbers

// paged_append_s4.hip
struct PagedAppend4 {
  const void *key, *value, *query;                        // query may be null
  long long k_row, k_head, v_row, v_head, q_row, q_head;  // elements
  void* q_out;                                            // [rows, q_heads, D] packed
  int q_heads, q_type;                                    // PT_S8, PT_F16 or PT_BF16
  const float* cos_sin;
  int rot, positions;
  bool neighbours, fill;
  float alpha_q, alpha_k, alpha_v;
};
int launch_paged_kv_append_s4(int type, const PagedAppend4& a, const PagedCache4& c, const PagedBatch& b, hipStream_t stream);
struct PagedRead4 {
  void *key, *value;  // [rows, heads, D] packed
  bool fill;
  float alpha_k, alpha_v;
};
int launch_paged_kv_read_s4(int type, const PagedRead4& a, const PagedCache4& c, const PagedBatch& b, hipStream_t stream);

// paged_attn_s4.hip
struct PagedAttn4 {
  const void* q;
  long long q_row, q_head;  // elements
  int q_heads, q_type;      // PT_S8, PT_F16 or PT_BF16
  void* out;                // [rows, q_heads, D] packed
  float alpha_qk, alpha_pv;
  int window, sinks;  // keys that a token sees, its own counted (0: all), and first keys that it sees beside them
  bool fill;
  int* arrivals;
  long long arrivals_count;
};
long long paged_attn_s4_arrivals(long long rows, long long seqs, long long q_heads, long long kv_heads, long long capacity);
long long paged_attn_s4_workspace_bytes(long long rows, long long seqs, long long q_heads, long long kv_heads, long long D,
                                        long long capacity);
int launch_paged_attn_s4(int out_type, const PagedAttn4& a, const PagedCache4& c, const PagedBatch& b, void* workspace,
                         long long workspace_bytes, hipStream_t stream);

}  // namespace ti
