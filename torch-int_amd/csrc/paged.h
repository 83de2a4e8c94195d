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
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int page_shift, int i) {
  PagedSeq s;
  const int cap = b.per_seq << page_shift;
  int lo = b.cu[i], hi = b.cu[i + 1];
  lo = lo < 0 ? 0 : lo > b.rows ? b.rows : lo;
  hi = hi < lo ? lo : hi > b.rows ? b.rows : hi;
  const int len = b.lens[i];
  s.row0 = lo;
  s.T = hi - lo;
  s.end = len < 0 ? 0 : len < (1 << 30) ? len : 1 << 30;
  s.len = s.end > cap ? cap : s.end;
  return s;
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

}  // namespace ti
