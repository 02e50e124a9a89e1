// The paged KV cache: argument blocks, page layout and the addressing shared
// by its writes, its reads (paged_cache.hip) and the attention over it
// (paged_attn.hip).
#pragma once

#include "common.hpp"

// Argument blocks (the layout of include/mtplx_amd.h).
struct mtp_rotary_args {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const int32_t* positions;
  const void* table;
  int T, Hq, Hkv, D, dims, traditional;
  float gain;
  long long q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head;
};

struct mtp_head_args {
  const void* q_weight;
  const void* k_weight;
  const int32_t* positions;
  long long axis0, axis1, axis2, axis3;
  int axes;
  float eps;
};

struct mtp_paged_write_args {
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  const void* table;
  void* k_pages;
  void* v_pages;
  void* k_scales;
  void* v_scales;
  const int32_t* block_table;
  const int32_t* q_start;
  const int32_t* row_off;
  int32_t* status;
  int T, B, width, Hq, Hkv, D, page_size, num_pages, bits, dims, traditional, max_rows;
  float gain;
  long long k_token, k_head, v_token, v_head, q_token, q_head, qo_token, qo_head;
};

struct mtp_paged_read_args {
  const void* k_pages;
  const void* v_pages;
  const void* k_scales;
  const void* v_scales;
  const int32_t* block_table;
  const int32_t* start;
  const int32_t* lengths;
  void* k_out;
  void* v_out;
  int32_t* status;
  int B, width, count, Hkv, D, page_size, num_pages, bits;
};

struct mtp_paged_attn_args {
  const void* q;
  void* out;
  const void* k_pages;
  const void* v_pages;
  const void* k_scales;
  const void* v_scales;
  const int32_t* block_table;
  const int32_t* q_start;
  const int32_t* row_off;
  int32_t* status;
  void* ws;
  size_t ws_bytes;
  int T, B, width, Hq, Hkv, D, page_size, num_pages, bits, max_rows;
  float scale;
  long long q_token, q_head, out_token, out_head;
};

struct mtp_attn_scope {
  int window, sinks, shared;
};

namespace mtp {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Pages hold [Hkv][page_size / 32] blocks of 32 keys x D, each in the order
// in which an attention wave loads its v_mfma_f32_32x32x16_bf16 operands: 64
// lanes x 16 contiguous bytes, so an operand is one 1 KB load and V needs no
// transposition when it is read. With h2 the half of D (K) and of every eight
// keys (V) that lane group l / 32 takes:
//   16 bits  K: d = (D/2) h2 + 8 i + e            at ((2 i + h2) 32 + key) 8 + e
//            V: d = 32 t + c, key = 16 jj + r,
//               r = 4 h2 + e (e < 4), 8 + 4 h2 + e - 4   at ((2 t + jj) 64 + 32 h2 + c) 8 + e
//   8 bits   two operands to a lane's 16 bytes:
//            K: d = (D/2) h2 + 16 i + e           at ((2 i + h2) 32 + key) 16 + e
//            V: as above                          at ((t 64) + 32 h2 + c) 16 + 8 jj + e
// At D = 128 and 16 bits these are the verify step's own blocks (kblk_index,
// vblk_index).
constexpr int kBlk = 32;   // keys of a block

template <int D, int BITS>
__device__ __forceinline__ int page_k_index(int key, int d) {
  constexpr int CH = BITS == 8 ? 16 : 8;
  const int h2 = d / (D / 2), dd = d % (D / 2);
  return (((dd / CH) * 2 + h2) * 32 + key) * CH + dd % CH;
}

// Key (of 16) in slot e (of 8) of lane half h2.
__device__ __forceinline__ int v_slot_key(int h2, int e) { return e < 4 ? 4 * h2 + e : 4 + 4 * h2 + e; }

// And the half and the slot of a key of 16.
__device__ __forceinline__ int v_key_half(int k) { return (k >> 2) & 1; }
__device__ __forceinline__ int v_key_slot(int k) { return (k & 3) + (k >> 3) * 4; }
template <int D, int BITS>
__device__ __forceinline__ int page_v_index(int key, int d) {
  const int lane = 32 * v_key_half(key & 15) + d % 32, e = v_key_slot(key & 15);
  return BITS == 8 ? (d / 32 * 64 + lane) * 16 + 8 * (key >> 4) + e : ((2 * (d / 32) + (key >> 4)) * 64 + lane) * 8 + e;
}

// The same value, computed here: what follows from it is not kept in registers
// across a loop (a spill's reload waits for every load in flight).
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// a / b of a >= 0, b > 0; 32-bit division where that does.
__device__ __forceinline__ long long div_pos(long long a, int b) {
  return a >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// Status bits: a position outside the block table (or a page outside the
// pool) was asked for; that row was not written, or reads as absent.
constexpr int kStatusPage = 1;

// Keys [lo, hi) of the block from position `base` on that lie in [from, to).
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange block_keys(long long base, long long from, long long to) {
  const long long a = from - base, b = to - base;
  return {a < 0 ? 0 : a < kBlk ? (int)a : kBlk, b < 0 ? 0 : b < kBlk ? (int)b : kBlk};
}

// First element of block `blk` (of a request's positions) of head h, or -1
// where the table holds no page of the pool for it.
__device__ __forceinline__ long long page_block(const int32_t* table, int width, int b, long long blk, int bpp,
                                                int num_pages, int Hkv, int h, int elems) {
  if (blk < 0 || blk >= (long long)width * bpp) return -1;
  const uint32_t page = (uint32_t)blk / (uint32_t)bpp;   // (width * page_size < 2^31)
  const int id = table[(size_t)b * width + page];
  if (id < 0 || id >= num_pages) return -1;
  return (((long long)id * Hkv + h) * bpp + (int)((uint32_t)blk - page * (uint32_t)bpp)) * elems;
}

// Rows [lo, hi) of the packed tokens that belong to request b, whatever the
// device array holds: never outside [0, T).
struct ReqRows {
  int lo, n;
};
__device__ __forceinline__ ReqRows req_rows(const int32_t* row_off, int b, int B, int T) {
  int lo, hi;
  if (row_off) {
    lo = row_off[b];
    hi = row_off[b + 1];
    lo = lo < 0 ? 0 : (lo > T ? T : lo);
    hi = hi > T ? T : hi;
  } else {
    const int L = T / B;
    lo = b * L;
    hi = lo + L;
  }
  return {lo, hi > lo ? hi - lo : 0};
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Checks that the entry points over pages share.
inline int check_pages(const char* who, int D, int page_size, int num_pages, int width, int bits, int B, int Hkv) {
  if (D != 64 && D != 128 && D != 256) {
    set_error("%s: head_dim %d unsupported (64, 128 or 256)", who, D);
    return MTP_ERR_UNSUPPORTED;
  }
  if (bits != 8 && bits != 16) {
    set_error("%s: %d-bit pages unsupported (8 or 16)", who, bits);
    return MTP_ERR_UNSUPPORTED;
  }
  if (page_size < 32 || page_size % 32 || num_pages < 1 || width < 1 || B < 1 || Hkv < 1 ||
      (long long)width * page_size > 0x7fffffffLL) {
    set_error("%s: bad page_size=%d num_pages=%d width=%d B=%d Hkv=%d (pages of a positive multiple of 32 keys, "
              "width * page_size < 2^31)", who, page_size, num_pages, width, B, Hkv);
    return MTP_ERR_ARG;
  }
  return MTP_OK;
}

inline bool row_strides(long long token, long long head, int D) {
  return token >= 0 && head >= D && token % 8 == 0 && head % 8 == 0;
}

}  // namespace mtp
