// Geometry of the paged key/value cache, shared by the append, read and
// attention kernels.
//
// The pool holds `pages` pages of [Hk][head bytes]; the bytes of one head of a
// page are its keys, then its values.  With S tokens a page, D values a head
// and NG = D / 32 groups:
//   XM_KV_F16   [S][D] fp16 each
//   XM_KV_Q4_0  [S][D / 2] bytes of codes, then [S][NG] fp16 scales, each; a
//               group of 32 values is d (c - 8), the values of a GGUF Q4_0
//               block.
// Order of the codes in a row, chosen so that the fragments of the attention's
// matrix instructions come out of whole 32-bit words by masks alone:
//   keys    word p (32 bits): nibble i is value 32 (p % NG) + 8 (p / NG) + i
//           (the NG words of a quarter of every group are one wide load)
//   values  halfword h (16 bits): nibble i is value 32 (h % NG) + 4 (h / NG) + i
//           (the D / 8 nibbles of one eighth of every group are one wide load)
//
// A call names its new tokens by rows: row t belongs to the sequence s with
// cu[s] <= t < cu[s + 1] (cu null: row t is sequence t), and sits at position
// lens[s] - (cu[s + 1] - t).  Position p of sequence s is slot p % S of page
// table[s][p / S].
#pragma once

#include "xm_gemv_dot.cuh"

struct KvView {
  uint8_t* pool;
  int64_t pages;
  int64_t head_bytes;      // K and V of one head of a page
  const int* table;
  int64_t table_stride;
  int table_width;         // entries of a row
  const int* cu;
  const int* lens;
  int B;
  int Hk;
  int page_shift;          // log2(tokens per page)
};

// Bytes of the keys (or of the values) of one head of a page.
__host__ __device__ inline int64_t kv_part_bytes(int kv_type, int D, int page_size) {
  return kv_type == XM_KV_F16 ? (int64_t)page_size * D * 2 : (int64_t)page_size * (D / 2 + D / 16);
}

// The sequence and position of row t (position negative: the sequence holds fewer tokens than it has
// rows; sequence -1: behind the last one).  Every lane of the warp calls it with the same t: the offsets are
// compared 32 at a time, so that their loads do not wait for one another.
struct KvPlace {
  int seq;
  int64_t pos;
};
XM_DEV KvPlace kv_place(const KvView& kv, int64_t t) {
  if (!kv.cu) return t < kv.B ? KvPlace{(int)t, (int64_t)__ldg(kv.lens + t) - 1} : KvPlace{-1, -1};
  const int lane = threadIdx.x & 31;
  int seq = 0;
#pragma unroll 4
  for (int s0 = 0; s0 < kv.B; s0 += 32) {             // how many sequences end at or before t
    const bool past = s0 + lane < kv.B && (int64_t)__ldg(kv.cu + s0 + lane + 1) <= t;
    seq += __popc(__ballot_sync(0xffffffffu, past));
  }
  if (seq >= kv.B || (int64_t)__ldg(kv.cu + seq) > t) return KvPlace{-1, -1};
  return KvPlace{seq, (int64_t)__ldg(kv.lens + seq) - ((int64_t)__ldg(kv.cu + seq + 1) - t)};
}

// The page that holds position pos >= 0 of sequence s, or -1 (and the error bit) where the table or
// the pool has no such page.
XM_DEV int64_t kv_page(const KvView& kv, int s, int64_t pos) {
  const int64_t slot = pos >> kv.page_shift;
  if (slot < kv.table_width) {
    const int page = __ldg(kv.table + (int64_t)s * kv.table_stride + slot);
    if (page >= 0 && page < kv.pages) return page;
  }
  atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
  return -1;
}
