// Rotary positions of packed tokens, and the paged KV cache's writes (rotating
// and quantising on the way) and reads. All of them move bytes once, and long
// calls are bound by that (a large copy reaches 5.17 TB/s on an MI355X):
//
//   rotation of 8192 tokens, 40 + 8 heads of 128: 46 us (201 MB, 4.4 TB/s);
//   write of the same at 8 bits, queries rotated: 58 us (218 MB, 3.8 TB/s);
//   its read back: 11 us (50 MB); eight requests' prefixes: 74 us (349 MB, 4.7).
//
// Writes and reads go by blocks of 32 positions of one head. A wave has a block
// to itself (writes: K or V of it, reads both): 8 or 16 KB of loads are under
// way before it waits, and nothing waits for another wave. With a workgroup of
// four waves and barriers per block the same calls took 75, 15 and 103 us.
// V's transposition is done on 32-bit words of LDS rows (two bf16 or four
// bytes of a key) and byte permutes, not element by element.
#include "paged.hpp"
#include "rotary.hpp"

namespace mtp {

constexpr int kNT = 256;

struct RotRows {
  const uint16_t* src;
  uint16_t* dst;
  long long st, sh, dt, dh;   // token and head strides in elements
};

// Tokens [t0, t0 + n) of the rows, every head of q and then of k, by the whole
// workgroup; cs [n][dims / 2].
__device__ __forceinline__ void rotate_rows(const RotRows& q, int Hq, const RotRows& k, int Hkv, int t0, int n, int D,
                                            const RotSpec& r, const float2* cs) {
  const int ipr = rot_items(D, r.dims, r.trad), heads = Hq + Hkv, half = r.dims / 2;
  const int total = n * heads * ipr;
  for (int x = threadIdx.x; x < total; x += kNT) {
    const int it = x % ipr, th = x / ipr;
    const int h = th % heads, t = th / heads;
    const bool isq = h < Hq;
    const RotRows& s = isq ? q : k;
    const int hh = isq ? h : h - Hq;
    uint16_t* dst = s.dst + (t0 + t) * s.dt + hh * s.dh;
    rot_item(it, s.src + (t0 + t) * s.st + hh * s.sh, r.dims, r.trad, [&](int i) { return cs[t * half + i]; },
             [&](int d, uint4 v) { *reinterpret_cast<uint4*>(dst + d) = v; });
  }
}

// A workgroup rotates up to eight tokens, all heads of each: the angles are
// computed once per token (64 pairs, not 48 heads x 64) and stay in LDS.
constexpr int kRotTokens = 8;    // most tokens of a workgroup
constexpr int kMaxPairs = 128;   // head dim 256 at most

__global__ __launch_bounds__(kNT) void rotary_kernel(RotRows q, RotRows k, const int32_t* positions, int T, int Hq,
                                                     int Hkv, int D, RotSpec r, int tokens) {
  __shared__ float2 cs[kRotTokens * kMaxPairs];
  const int half = r.dims / 2;
  for (long long t0 = (long long)blockIdx.x * tokens; t0 < T; t0 += (long long)gridDim.x * tokens) {
    const int n = T - t0 < tokens ? (int)(T - t0) : tokens;
    for (int x = threadIdx.x; x < n * half; x += kNT)
      cs[x] = rot_angle(positions[t0 + x / half], r.table[x % half], r.gain);
    __syncthreads();
    rotate_rows(q, Hq, k, Hkv, (int)t0, n, D, r, cs);
    __syncthreads();
  }
}

struct WriteParams {
  const uint16_t* k;
  const uint16_t* v;
  unsigned char* k_pages;
  unsigned char* v_pages;
  float* k_scales;
  float* v_scales;
  const int32_t* block_table;
  const int32_t* q_start;
  const int32_t* row_off;
  int32_t* status;
  int T, B, width, Hkv, bpp, num_pages;
  long long k_token, k_head, v_token, v_head;
  RotSpec r;
  RotRows q;
  int Hq, q_tokens, kv_groups;   // workgroups [0, kv_groups) write K and V, the others rotate q
  int nb_uniform;                // blocks of each request where row_off is null
};

__device__ __forceinline__ long long floor_blk(long long p) { return p >> 5; }   // (blocks of 32)

// Blocks of 32 positions that request b's new tokens fall into, from the
// block of the first one on.
__device__ __forceinline__ int touched_blocks(long long start, int n) {
  return n > 0 ? (int)(floor_blk(start + n - 1) - floor_blk(start)) + 1 : 0;
}

// A wave's work: one block of 32 positions of one request, one head, K or V.
struct Unit {
  ReqRows rows;
  long long start, blk;   // first position of the request, block of positions
  int b;
};

// Unit u (of one head) of the call. With row offsets every wave scans the
// requests' block counts, 64 at a time. False behind the last one.
__device__ __forceinline__ bool find_unit(const WriteParams& p, long long u, int lane, Unit& w) {
  if (!p.row_off) {
    if (u >= (long long)p.B * p.nb_uniform) return false;
    w.b = (int)div_pos(u, p.nb_uniform);
    w.rows = req_rows(nullptr, w.b, p.B, p.T);
    w.start = p.q_start[w.b];
    w.blk = floor_blk(w.start) + (u - (long long)w.b * p.nb_uniform);
    return true;
  }
  long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int bb = b0 + lane;
    ReqRows r = {0, 0};
    int start = 0, cnt = 0;
    if (bb < p.B) {
      r = req_rows(p.row_off, bb, p.B, p.T);
      start = p.q_start[bb];
      cnt = touched_blocks(start, r.n);
    }
    int incl = cnt;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(incl, off, 64);
      if (lane >= off) incl += t;
    }
    const unsigned long long m = __ballot(u < carry + incl);   // the first whose end lies behind u
    if (m) {
      const int src = __ffsll((long long)m) - 1;
      w.b = __builtin_amdgcn_readfirstlane(b0 + src);
      w.rows.lo = __builtin_amdgcn_readlane(r.lo, src);
      w.rows.n = __builtin_amdgcn_readlane(r.n, src);
      w.start = __builtin_amdgcn_readlane(start, src);
      w.blk = floor_blk(w.start) + (int)(u - carry) - __builtin_amdgcn_readlane(incl - cnt, src);
      return true;
    }
    carry += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// What a wave's lanes left in LDS is there for its other lanes (one wave's LDS
// accesses complete in order; this keeps the compiler's order).
__device__ __forceinline__ void wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// LDS of a wave: 32 rows, padded so that 16-byte accesses of 8 rows hit
// distinct banks; 8-bit rows take their place.
template <int D>
constexpr int row16() { return D + 8; }    // elements
template <int D>
constexpr int row8() { return D + 16; }    // bytes
template <int D>
constexpr int cache_waves() { return D == 256 ? 2 : 4; }

// Lane l's half (l / 32) of row l % 32.
template <int D>
__device__ __forceinline__ void half_row(const uint16_t* rows, int lane, u32x4 (&x)[D / 16]) {
  const uint16_t* row = rows + (lane & 31) * row16<D>() + (lane >> 5) * (D / 2);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) x[i] = reinterpret_cast<const u32x4*>(row)[i];
}

// 8-bit rows. Largest magnitude A, by the bits of bf16 (m: of each two
// elements); then A / 127 and r = 127 (1 / A), each step rounded once, and
// q = rint(x r): adding 1.5 2^23 rounds to an integer in the low bits,
// |x r| < 127.5. (The reciprocal first, as torch computes 127 / A on the GPU:
// ratios of short mantissas often lie halfway between integers, and rows
// quantised there and here then hold the same ones.) A row with a NaN or an infinity gets a NaN scale, so it
// reads as NaN instead of as wrong numbers; one below 2^-100 gets zeros
// (r would overflow, A / 127 go subnormal).
__device__ __forceinline__ u16x2 max_bits(u16x2 m, u32x4 x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[j] & 0x7fff7fffu));
  return m;
}
struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(int m) {
  const float a = __uint_as_float((uint32_t)m << 16);
  const bool bad = m >= 0x7f80, tiny = a < 0x1p-100f;
  return {bad || tiny ? 0.f : __fmul_rn(127.f, 1.f / a), bad ? __uint_as_float(0x7fc00000u) : tiny ? 0.f : a / 127.f};
}
__device__ __forceinline__ uint2 bytes8(u32x4 x, float inv) {
#pragma clang fp contract(off)   // (the product is rounded before the sum)
  const Chunk8 c = unpack8(__builtin_bit_cast(uint4, x));
  uint32_t q[8];   // (NaN has zeros in its low byte)
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = __float_as_uint(c.v[j] * inv + 12582912.f);
  return make_uint2(__builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu),
                    __builtin_amdgcn_perm(q[5], q[4], 0x0c0c0400u) | __builtin_amdgcn_perm(q[7], q[6], 0x04000c0cu));
}

// Lane l's half row (half_row) as bytes; the row's scale, in both its lanes.
template <int D>
__device__ __forceinline__ float quantise(const u32x4 (&x)[D / 16], uint32_t (&w)[D / 8]) {
  u16x2 mx = {0, 0};
#pragma unroll
  for (int i = 0; i < D / 16; ++i) mx = max_bits(mx, x[i]);
  int m = mx.x > mx.y ? mx.x : mx.y;
  const int other = __shfl_xor(m, 32, 64);
  const RowScale s = row_scale(m > other ? m : other);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint2 q = bytes8(x[i], s.inv);
    w[2 * i] = q.x;
    w[2 * i + 1] = q.y;
  }
  return s.scale;
}

// Bytes j of four words, as the j-th word.
__device__ __forceinline__ void turn4(const uint32_t (&a)[4], uint32_t (&t)[4]) {
  const uint32_t lo01 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);
  const uint32_t lo23 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
  t[0] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
  t[1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
  t[2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
  t[3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
}

// Keys [klo, khi) of a block, few of them (a decode or verify step's): a lane
// has one 16-byte chunk of a row, its elements go where they belong. Up to two
// rounds of it; as whole blocks through LDS a decode step of sixteen requests
// took 10.4 us, this way 5.7 (6.8 with fp64 angles).
template <int D, int BITS>
__device__ __forceinline__ void write_few(const WriteParams& p, int h, bool isk, int lane, long long base,
                                          long long first, long long at, int klo, int khi) {
  constexpr int CPR = D / 8;   // lanes of a row
  const int dims = p.r.dims;
  const bool paired = rot_paired(dims, p.r.trad);
#pragma unroll 1
  for (int k0 = klo; k0 < khi; k0 += 64 / CPR) {
    lane = fresh(lane);
    const int c = lane % CPR, key = k0 + lane / CPR;
    const bool mine = key < khi;
    const long long token = first + (mine ? key : khi - 1);
    const int pos = (int)(base + key);
    const uint16_t* row = isk ? p.k + h * p.k_head + token * p.k_token : p.v + h * p.v_head + token * p.v_token;
    u32x4 x;
    auto angles = [&](int i) { return rot_angle(pos, p.r.table[i], p.r.gain); };
    if (isk && paired && 8 * c < dims) {
      const int half = dims / 2, d = 8 * c < half ? 8 * c : 8 * c - half;
      const Chunk8 a = unpack8(*reinterpret_cast<const uint4*>(row + d));
      const Chunk8 b = unpack8(*reinterpret_cast<const uint4*>(row + d + half));
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 w = angles(d + e);
        y[e] = 8 * c < half ? rot_first(a.v[e], b.v[e], w) : rot_second(a.v[e], b.v[e], w);
      }
      x = __builtin_bit_cast(u32x4, pack8(y));
    } else if (isk && !paired && 8 * c < dims) {
      rot_item(c, row, dims, p.r.trad, angles, [&](int, uint4 v) { x = __builtin_bit_cast(u32x4, v); });
    } else {
      x = *reinterpret_cast<const u32x4*>(row + 8 * c);
    }
    unsigned char* dst = (isk ? p.k_pages : p.v_pages) + (size_t)at * (BITS / 8);
    if constexpr (BITS == 16) {
      if (!mine) continue;
      if (isk) {
        *reinterpret_cast<u32x4*>(dst + 2 * page_k_index<D, BITS>(key, 8 * c)) = x;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          reinterpret_cast<uint16_t*>(dst)[page_v_index<D, BITS>(key, 8 * c + e)] = (uint16_t)(x[e / 2] >> (16 * (e & 1)));
      }
    } else {
      const u16x2 mx = max_bits(u16x2{0, 0}, x);
      int m = mx.x > mx.y ? mx.x : mx.y;
#pragma unroll
      for (int off = 1; off < CPR; off <<= 1) {
        const int o = __shfl_xor(m, off, 64);
        m = m > o ? m : o;
      }
      const RowScale s = row_scale(m);
      const uint2 q = bytes8(x, s.inv);
      if (!mine) continue;
      if (c == 0) ((isk ? p.k_scales : p.v_scales) + at / D)[key] = s.scale;   // [page][head][slot]
      if (isk) {
        *reinterpret_cast<uint2*>(dst + page_k_index<D, BITS>(key, 8 * c)) = q;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dst[page_v_index<D, BITS>(key, 8 * c + e)] = (unsigned char)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
      }
    }
  }
}

// One unit by one wave, in its own LDS: rows come whole, turn in LDS and leave
// in the page's order, 16 bytes a lane; keys of a block that is not all new go
// out element by element (V) or chunk by chunk (K).
template <int D, int BITS>
__device__ __forceinline__ void write_unit(const WriteParams& p, const Unit& w, int h, bool isk, int lane,
                                           uint16_t* rows) {
  constexpr int RS = row16<D>(), NC = D / 16, BS = row8<D>();   // 16-byte loads of a lane
  const long long base = w.blk * kBlk;
  // Keys [klo, khi) of the block are new; token of key kk: first + kk.
  const KeyRange range = block_keys(base, w.start, w.start + w.rows.n);
  const int klo = range.lo, khi = range.hi;
  if (klo >= khi) return;   // (a request of no rows)
  const long long first = w.rows.lo + (base - w.start);
  u32x4 x[NC];
  const bool few = khi - klo <= 1024 / D;
  if (!few) {
    const uint16_t* src = isk ? p.k + h * p.k_head : p.v + h * p.v_head;
    const long long st = isk ? p.k_token : p.v_token;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = i * 64 + lane;
      int kk = c / (D / 8);
      kk = kk < klo ? klo : kk >= khi ? khi - 1 : kk;   // (other keys' rows: the nearest new one's)
      x[i] = *reinterpret_cast<const u32x4*>(src + (first + kk) * st + c % (D / 8) * 8);
    }
  }
  const long long at = page_block(p.block_table, p.width, w.b, w.blk, p.bpp, p.num_pages, p.Hkv, h, kBlk * D);
  if (at < 0) {
    if (p.status && lane == 0) atomicOr(p.status, kStatusPage);
    return;
  }
  if (few) {
    write_few<D, BITS>(p, h, isk, lane, base, first, at, klo, khi);
    return;
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = i * 64 + lane;
    *reinterpret_cast<u32x4*>(rows + c / (D / 8) * RS + c % (D / 8) * 8) = x[i];
  }
  wave_lds();
  unsigned char* dst = (isk ? p.k_pages : p.v_pages) + (size_t)at * (BITS / 8);
  const int key = lane & 31;
  const bool mine = key >= klo && key < khi;   // the lane's row
  if (isk && p.r.dims) {   // in place: an item reads what it stores, or the source
    const int np = rot_paired(p.r.dims, p.r.trad) ? p.r.dims / 16 : (p.r.dims + 7) / 8;
    const bool inplace = p.r.trad || rot_paired(p.r.dims, p.r.trad);
    for (int x = lane; x < 32 * np; x += 64) {
      const int kk = x / np;
      if (kk < klo || kk >= khi) continue;
      const int pos = (int)(base + kk);
      uint16_t* row = rows + kk * RS;
      auto angles = [&](int i) { return rot_angle(pos, p.r.table[i], p.r.gain); };
      auto store = [&](int d, uint4 v) { *reinterpret_cast<uint4*>(row + d) = v; };
      if (inplace)
        rot_item(x % np, row, p.r.dims, p.r.trad, angles, store);
      else
        rot_item(x % np, p.k + h * p.k_head + (first + kk) * p.k_token, p.r.dims, p.r.trad, angles, store);
    }
    wave_lds();
  }
  uint32_t q[D / 8];   // 8 bits: the lane's half row
  if constexpr (BITS == 8) {
    half_row<D>(rows, lane, x);
    const float s = quantise<D>(x, q);
    if (mine && lane < 32) ((isk ? p.k_scales : p.v_scales) + at / D)[key] = s;   // [page][head][slot]
  }
  if (isk) {
    if constexpr (BITS == 16) half_row<D>(rows, lane, x);
    if (mine) {
      if constexpr (BITS == 16) {
#pragma unroll
        for (int i = 0; i < NC; ++i) *reinterpret_cast<u32x4*>(dst + (i * 64 + lane) * 16) = x[i];
      } else {
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
          *reinterpret_cast<u32x4*>(dst + (i * 64 + lane) * 16) = u32x4{q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]};
      }
    }
    wave_lds();
    return;
  }
  const bool all = klo == 0 && khi == kBlk;
  if constexpr (BITS == 16) {
    if (all) {
#pragma unroll
      for (int i = 0; i < 2 * D / 64; ++i) {   // two columns, the eight keys of a chunk each
        const int x = i * 64 + lane, c = x % 16 * 2, hh = (x >> 4) & 1, tj = x >> 5;
        const uint16_t* col = rows + 16 * (tj & 1) * RS + 32 * (tj >> 1) + c;
        uint32_t a[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = *reinterpret_cast<const uint32_t*>(col + v_slot_key(hh, e) * RS);
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = __builtin_amdgcn_perm(a[2 * e + 1], a[2 * e], 0x05040100u);
          hi[e] = __builtin_amdgcn_perm(a[2 * e + 1], a[2 * e], 0x07060302u);
        }
        u32x4* to = reinterpret_cast<u32x4*>(dst) + tj * 64 + hh * 32 + c;
        to[0] = u32x4{lo[0], lo[1], lo[2], lo[3]};
        to[1] = u32x4{hi[0], hi[1], hi[2], hi[3]};
      }
    } else {
      for (int x = lane; x < (khi - klo) * D; x += 64) {
        const int kk = klo + x / D, d = x % D;
        reinterpret_cast<uint16_t*>(dst)[page_v_index<D, 16>(kk, d)] = rows[kk * RS + d];
      }
    }
  } else {
    wave_lds();
    unsigned char* bytes = reinterpret_cast<unsigned char*>(rows);
#pragma unroll
    for (int i = 0; i < NC / 2; ++i)
      *reinterpret_cast<u32x4*>(bytes + key * BS + (lane >> 5) * (D / 2) + 16 * i) =
          u32x4{q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]};
    wave_lds();
    if (all) {
      for (int x = lane; x < D / 2; x += 64) {   // four columns, the sixteen keys of a chunk each
        const int c = x % 8 * 4, hh = (x >> 3) & 1, t = x >> 4;
        uint32_t o[4][4];   // [keys][column]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            a[e] = *reinterpret_cast<const uint32_t*>(bytes + (16 * (j >> 1) + v_slot_key(hh, 4 * (j & 1) + e)) * BS + 32 * t + c);
          turn4(a, o[j]);
        }
        u32x4* to = reinterpret_cast<u32x4*>(dst) + t * 64 + hh * 32 + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = u32x4{o[0][e], o[1][e], o[2][e], o[3][e]};
      }
    } else {
      for (int x = lane; x < (khi - klo) * D; x += 64) {
        const int kk = klo + x / D, d = x % D;
        dst[page_v_index<D, 8>(kk, d)] = bytes[kk * BS + d];
      }
    }
  }
  wave_lds();
}

// Request of packed token t: the b with row_off[b] <= t < row_off[b + 1], or
// -1 behind the last one; position in *pos.
__device__ __forceinline__ int token_request(const WriteParams& p, int t, long long* pos) {
  int b = 0;
  if (p.row_off) {
    int lo = 0, hi = p.B;   // the last b with row_off[b] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.row_off[mid] <= t) lo = mid; else hi = mid;
    }
    b = lo;
  } else {
    b = t / (p.T / p.B);
  }
  const ReqRows rq = req_rows(p.row_off, b, p.B, p.T);
  if (t < rq.lo || t >= rq.lo + rq.n) return -1;
  *pos = (long long)p.q_start[b] + (t - rq.lo);
  return b;
}

template <int D, int BITS>
__global__ __launch_bounds__(64 * cache_waves<D>(), D == 256 ? 1 : 4) void paged_write_kernel(WriteParams p) {
  constexpr int NT = 64 * cache_waves<D>();
  __shared__ __attribute__((aligned(16))) uint16_t lds[cache_waves<D>()][32 * row16<D>()];
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x >= p.kv_groups) {   // rotate queries, q_tokens at a time
    float2* cs = reinterpret_cast<float2*>(&lds[0][0]);
    __shared__ int s_live[kRotTokens];
    const int half = p.r.dims / 2, ipr = rot_items(D, p.r.dims, p.r.trad);
    const int stride = ((int)gridDim.x - p.kv_groups) * p.q_tokens;
    for (int t0 = ((int)blockIdx.x - p.kv_groups) * p.q_tokens; t0 < p.T; t0 += stride) {
      const int n = p.T - t0 < p.q_tokens ? p.T - t0 : p.q_tokens;
      for (int t = 0; t < n; ++t) {
        long long pos = 0;
        const int b = token_request(p, t0 + t, &pos);   // the same in every thread
        if (threadIdx.x == 0) s_live[t] = b >= 0;
        for (int x = threadIdx.x; x < half; x += NT) cs[t * half + x] = rot_angle(pos, p.r.table[x], p.r.gain);
      }
      __syncthreads();
      for (int x = threadIdx.x; x < n * p.Hq * ipr; x += NT) {
        const int it = x % ipr, th = x / ipr;
        const int h = th % p.Hq, t = th / p.Hq;
        if (!s_live[t]) continue;   // rows behind the last request stay as they are
        uint16_t* dst = p.q.dst + (t0 + t) * p.q.dt + h * p.q.dh;
        rot_item(it, p.q.src + (t0 + t) * p.q.st + h * p.q.sh, p.r.dims, p.r.trad,
                 [&](int i) { return cs[t * half + i]; },
                 [&](int d, uint4 v) { *reinterpret_cast<uint4*>(dst + d) = v; });
      }
      __syncthreads();
      if (t0 > p.T - stride) break;   // (t0 + stride could pass 2^31)
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (long long x = (long long)blockIdx.x * cache_waves<D>() + wave;; x += (long long)p.kv_groups * cache_waves<D>()) {
    Unit w;
    const long long u = div_pos(x >> 1, p.Hkv);
    if (!find_unit(p, u, lane, w)) return;   // (no barrier follows)
    write_unit<D, BITS>(p, w, (int)((x >> 1) - u * p.Hkv), (x & 1) == 0, fresh(lane), lds[wave]);
  }
}

struct ReadParams {
  const unsigned char* k_pages;
  const unsigned char* v_pages;
  const float* k_scales;
  const float* v_scales;
  const int32_t* block_table;
  const int32_t* start;
  const int32_t* lengths;
  uint16_t* k_out;
  uint16_t* v_out;
  int32_t* status;
  int B, width, count, Hkv, bpp, num_pages, nb;
};

// One wave: a block of 32 positions of one request, one head, K and V, from the
// page's order through its LDS back into rows [B, Hkv, count, D]. 8-bit
// elements turn as bytes and are widened on their way out.
template <int D, int BITS>
__device__ __forceinline__ void read_unit(const ReadParams& p, int b, int h, int blk, int lane, unsigned char* lds) {
  constexpr int NC = D * BITS / 256;   // 16-byte loads of a lane
  constexpr int RS = BITS == 8 ? row8<D>() : row16<D>() * 2;   // bytes of a row
  constexpr bool AHEAD = NC <= 8;
  const long long start = p.start ? p.start[b] : 0;
  const long long ablk = floor_blk(start) + blk, base = ablk * kBlk;
  const KeyRange range = block_keys(base, start, start + p.count);
  const int klo = range.lo, khi = range.hi;
  if (klo >= khi) return;
  const long long len = p.lengths ? (long long)p.lengths[b] - base : kBlk;
  int live = len < khi ? (len < 0 ? 0 : (int)len) : khi;   // keys [klo, live) are read, [live, khi) are zeros
  if (live < klo) live = klo;
  long long at = -1;
  if (live > klo) {
    at = page_block(p.block_table, p.width, b, ablk, p.bpp, p.num_pages, p.Hkv, h, kBlk * D);
    if (at < 0) {
      if (p.status && lane == 0) atomicOr(p.status, kStatusPage);
      live = klo;
    }
  }
  constexpr int W = BITS == 8 ? 4 : 2, NV = NC < W ? W : NC;   // (D = 64, 8 bits: half the lanes hold all of V)
  u32x4 kx[NC], vx[NV];
  float ks = 0.f, vs = 0.f;   // lane l: key l % 32's
  auto ask = [&](u32x4 (&x)[NC], const unsigned char* pool) {
    const unsigned char* src = pool + (size_t)at * (BITS / 8);
#pragma unroll
    for (int i = 0; i < NC; ++i) x[i] = *reinterpret_cast<const u32x4*>(src + (i * 64 + lane) * 16);
  };
  // V's chunks by what turns together: four columns of 16 keys, or two of 8.
  auto ask_v = [&]() {
    const u32x4* src = reinterpret_cast<const u32x4*>(p.v_pages + (size_t)at * (BITS / 8));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int x = (i / W) * 64 + lane;
      const int c = BITS == 8 ? x / 8 * 32 + x % 8 * 4 : x / 16 * 32 + x % 16 * 2;
      if (x * W < D * BITS / 4) vx[i] = src[c + i % W];
    }
  };
  if (at >= 0) {
    ask(kx, p.k_pages);
    if (AHEAD) ask_v();
    if constexpr (BITS == 8) {
      ks = (p.k_scales + at / D)[lane & 31];
      vs = (p.v_scales + at / D)[lane & 31];
    }
  }
  auto leave = [&](uint16_t* dst, float s) {   // rows [klo, khi): whole 16-byte chunks
    dst += (((size_t)b * p.Hkv + h) * p.count) * D;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int c = i * 64 + lane, kk = c / (D / 8), d = c % (D / 8) * 8;
      u32x4 o;
      if constexpr (BITS == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(lds + kk * RS + d);
        const float sk = __shfl(s, kk, 64);
        float y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = __fmul_rn((float)(int8_t)(w.x >> (8 * e)), sk);
          y[e + 4] = __fmul_rn((float)(int8_t)(w.y >> (8 * e)), sk);
        }
        o = __builtin_bit_cast(u32x4, pack8(y));
      } else {
        o = *reinterpret_cast<const u32x4*>(lds + kk * RS + d * 2);
      }
      if (kk >= live) o = u32x4{0, 0, 0, 0};
      if (kk >= klo && kk < khi) *reinterpret_cast<u32x4*>(dst + (base + kk - start) * D + d) = o;
    }
    wave_lds();
  };
  if (at >= 0) {   // lane l: its half of row l % 32
#pragma unroll
    for (int i = 0; i < NC; ++i)
      *reinterpret_cast<u32x4*>(lds + (lane & 31) * RS + (lane >> 5) * (D * BITS / 16) + 16 * i) = kx[i];
    wave_lds();
  }
  leave(p.k_out, ks);
  if (at >= 0) {
    if (!AHEAD) ask_v();
    if constexpr (BITS == 8) {
#pragma unroll
      for (int i = 0; i < NV; i += 4) {
        const int x = i / 4 * 64 + lane, c = x % 8 * 4, hh = (x >> 3) & 1, t = x >> 4;
        if (x >= D / 2) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a[4] = {vx[i][j], vx[i + 1][j], vx[i + 2][j], vx[i + 3][j]};
          uint32_t o[4];
          turn4(a, o);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint32_t*>(lds + (16 * (j >> 1) + v_slot_key(hh, 4 * (j & 1) + e)) * RS + 32 * t + c) = o[e];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; i += 2) {
        const int x = i / 2 * 64 + lane, c = x % 16 * 2, hh = (x >> 4) & 1, tj = x >> 5;
        unsigned char* col = lds + 16 * (tj & 1) * RS + (32 * (tj >> 1) + c) * 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = vx[i][e], bb = vx[i + 1][e];
          *reinterpret_cast<uint32_t*>(col + v_slot_key(hh, 2 * e) * RS) = __builtin_amdgcn_perm(bb, a, 0x05040100u);
          *reinterpret_cast<uint32_t*>(col + v_slot_key(hh, 2 * e + 1) * RS) = __builtin_amdgcn_perm(bb, a, 0x07060302u);
        }
      }
    }
    wave_lds();
  }
  leave(p.v_out, vs);
}

template <int D, int BITS>
__global__ __launch_bounds__(64 * cache_waves<D>()) void paged_read_kernel(ReadParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[cache_waves<D>()][32 * (BITS == 8 ? row8<D>() : row16<D>() * 2)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long units = (long long)p.B * p.Hkv * p.nb, step = (long long)gridDim.x * cache_waves<D>();
  for (long long u = (long long)blockIdx.x * cache_waves<D>() + wave; u < units; u += step) {
    const long long v = div_pos(u, p.nb), b = div_pos(v, p.Hkv);
    read_unit<D, BITS>(p, (int)b, (int)(v - b * p.Hkv), (int)(u - v * p.nb), lane, lds[wave]);
  }
}

inline int check_rotation(const char* who, const void* table, int dims, int D) {
  if (dims < 0 || dims > D || dims % 2 || (dims > 0 && !table)) {
    set_error("%s: dims=%d must be even, at most the head dim %d, and come with a table", who, dims, D);
    return MTP_ERR_ARG;
  }
  return MTP_OK;
}

// Tokens of a rotation workgroup: eight (one angle table for all their heads)
// once there is a workgroup for every CU that way, else fewer.
inline int rot_tokens(int T) { return T >= 8 * 256 ? 8 : T >= 4 * 256 ? 4 : T >= 2 * 256 ? 2 : 1; }

template <int D, int BITS>
void launch_write(const WriteParams& p, int groups, hipStream_t st) {
  hipLaunchKernelGGL((paged_write_kernel<D, BITS>), dim3((unsigned)groups), dim3(64 * cache_waves<D>()), 0, st, p);
}
template <int D, int BITS>
void launch_read(const ReadParams& p, int groups, hipStream_t st) {
  hipLaunchKernelGGL((paged_read_kernel<D, BITS>), dim3((unsigned)groups), dim3(64 * cache_waves<D>()), 0, st, p);
}

}  // namespace mtp

using namespace mtp;

MTP_API int mtp_rotary(const mtp_rotary_args* a, void* stream) {
  const char* who = "mtp_rotary";
  if (!a || !a->q || !a->q_out || !a->positions || a->T < 1 || a->Hq < 1 || a->Hkv < 0 || a->D < 8 || a->D % 8 ||
      a->D > 2 * kMaxPairs || (a->Hkv > 0 && (!a->k || !a->k_out))) {
    set_error("%s: bad arguments (D a multiple of 8 up to 256)", who);
    return MTP_ERR_ARG;
  }
  const int rc = check_rotation(who, a->table, a->dims, a->D);
  if (rc) return rc;
  if (!aligned16(a->q) || !aligned16(a->q_out) || !row_strides(a->q_token, a->q_head, a->D) ||
      !row_strides(a->qo_token, a->qo_head, a->D) ||
      (a->Hkv > 0 && (!aligned16(a->k) || !aligned16(a->k_out) || !row_strides(a->k_token, a->k_head, a->D) ||
                      !row_strides(a->ko_token, a->ko_head, a->D)))) {
    set_error("%s: rows must be 16-byte aligned, their strides multiples of 8 elements", who);
    return MTP_ERR_ARG;
  }
  const RotRows q = {(const uint16_t*)a->q, (uint16_t*)a->q_out, a->q_token, a->q_head, a->qo_token, a->qo_head};
  const RotRows k = {(const uint16_t*)a->k, (uint16_t*)a->k_out, a->k_token, a->k_head, a->ko_token, a->ko_head};
  const RotSpec r = {(const unsigned long long*)a->table, a->dims, a->traditional, a->gain};
  const int tokens = rot_tokens(a->T);
  const int groups = cdiv(a->T, tokens);
  hipLaunchKernelGGL(rotary_kernel, dim3((unsigned)groups), dim3(kNT), 0, (hipStream_t)stream, q, k, a->positions,
                     a->T, a->Hq, a->Hkv, a->D, r, tokens);
  return launch_check(who);
}

MTP_API int mtp_paged_write(const mtp_paged_write_args* a, void* stream) {
  const char* who = "mtp_paged_write";
  if (!a || !a->k || !a->v || !a->k_pages || !a->v_pages || !a->block_table || !a->q_start || a->T < 1 ||
      (a->bits == 8 && (!a->k_scales || !a->v_scales)) || (a->q && (!a->q_out || a->Hq < 1))) {
    set_error("%s: bad arguments", who);
    return MTP_ERR_ARG;
  }
  int rc = check_pages(who, a->D, a->page_size, a->num_pages, a->width, a->bits, a->B, a->Hkv);
  if (rc) return rc;
  rc = check_rotation(who, a->table, a->dims, a->D);
  if (rc) return rc;
  if (!a->row_off && a->T % a->B) {
    set_error("%s: %d tokens are no whole rows of %d requests (give row_off)", who, a->T, a->B);
    return MTP_ERR_ARG;
  }
  if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_pages) || !aligned16(a->v_pages) ||
      !row_strides(a->k_token, a->k_head, a->D) || !row_strides(a->v_token, a->v_head, a->D) ||
      (a->q && (!aligned16(a->q) || !aligned16(a->q_out) || !row_strides(a->q_token, a->q_head, a->D) ||
                !row_strides(a->qo_token, a->qo_head, a->D)))) {
    set_error("%s: rows must be 16-byte aligned, their strides multiples of 8 elements", who);
    return MTP_ERR_ARG;
  }
  WriteParams p = {};
  p.k = (const uint16_t*)a->k;
  p.v = (const uint16_t*)a->v;
  p.k_pages = (unsigned char*)a->k_pages;
  p.v_pages = (unsigned char*)a->v_pages;
  p.k_scales = (float*)a->k_scales;
  p.v_scales = (float*)a->v_scales;
  p.block_table = a->block_table;
  p.q_start = a->q_start;
  p.row_off = a->row_off;
  p.status = a->status;
  p.T = a->T;
  p.B = a->B;
  p.width = a->width;
  p.Hkv = a->Hkv;
  p.bpp = a->page_size / kBlk;
  p.num_pages = a->num_pages;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  p.r = {(const unsigned long long*)a->table, a->dims, a->traditional, a->gain};
  p.q = {(const uint16_t*)a->q, (uint16_t*)a->q_out, a->q_token, a->q_head, a->qo_token, a->qo_head};
  p.Hq = a->Hq;
  // n consecutive positions touch at most (n + 30) / 32 + 1 blocks; requests
  // of n_b rows, T in all, at most T / 32 + 2 B. The units are dealt round a
  // grid of that many workgroups, so max_rows only sizes it.
  const auto most = [](long long n) { return (n + 30) / kBlk + 1; };
  long long units;
  if (a->row_off) {
    units = (long long)a->T / kBlk + 2LL * a->B;
    if (a->max_rows > 0 && a->B * most(a->max_rows) < units) units = a->B * most(a->max_rows);
  } else {
    p.nb_uniform = (int)most(a->T / a->B);
    units = (long long)a->B * p.nb_uniform;
  }
  const int waves = a->D == 256 ? cache_waves<256>() : cache_waves<128>();
  long long groups = (units * 2 * a->Hkv + waves - 1) / waves;
  if (groups > 1 << 20) groups = 1 << 20;
  p.kv_groups = (int)groups;
  if (a->q) {
    p.q_tokens = rot_tokens(a->T);
    groups += cdiv(a->T, p.q_tokens) < (1 << 20) ? cdiv(a->T, p.q_tokens) : 1 << 20;
  }
  hipStream_t st = (hipStream_t)stream;
  const int key = a->D * 100 + a->bits;
  switch (key) {
    case 6416: launch_write<64, 16>(p, (int)groups, st); break;
    case 6408: launch_write<64, 8>(p, (int)groups, st); break;
    case 12816: launch_write<128, 16>(p, (int)groups, st); break;
    case 12808: launch_write<128, 8>(p, (int)groups, st); break;
    case 25616: launch_write<256, 16>(p, (int)groups, st); break;
    default: launch_write<256, 8>(p, (int)groups, st); break;
  }
  return launch_check(who);
}

MTP_API int mtp_paged_read(const mtp_paged_read_args* a, void* stream) {
  const char* who = "mtp_paged_read";
  if (!a || !a->k_pages || !a->v_pages || !a->block_table || !a->k_out || !a->v_out || a->count < 0 ||
      (a->bits == 8 && (!a->k_scales || !a->v_scales))) {
    set_error("%s: bad arguments", who);
    return MTP_ERR_ARG;
  }
  const int rc = check_pages(who, a->D, a->page_size, a->num_pages, a->width, a->bits, a->B, a->Hkv);
  if (rc) return rc;
  if (!aligned16(a->k_pages) || !aligned16(a->v_pages) || !aligned16(a->k_out) || !aligned16(a->v_out)) {
    set_error("%s: pages and outputs must be 16-byte aligned", who);
    return MTP_ERR_ARG;
  }
  if (a->count == 0) return MTP_OK;
  ReadParams p = {(const unsigned char*)a->k_pages, (const unsigned char*)a->v_pages, (const float*)a->k_scales,
                  (const float*)a->v_scales, a->block_table, a->start, a->lengths, (uint16_t*)a->k_out,
                  (uint16_t*)a->v_out, a->status, a->B, a->width, a->count, a->Hkv, a->page_size / kBlk,
                  a->num_pages, (int)(((long long)a->count + 30) / kBlk + 1)};
  const int waves = a->D == 256 ? cache_waves<256>() : cache_waves<128>();
  long long groups = ((long long)a->B * a->Hkv * p.nb + waves - 1) / waves;
  if (groups > 1 << 20) groups = 1 << 20;
  hipStream_t st = (hipStream_t)stream;
  switch (a->D * 100 + a->bits) {
    case 6416: launch_read<64, 16>(p, (int)groups, st); break;
    case 6408: launch_read<64, 8>(p, (int)groups, st); break;
    case 12816: launch_read<128, 16>(p, (int)groups, st); break;
    case 12808: launch_read<128, 8>(p, (int)groups, st); break;
    case 25616: launch_read<256, 16>(p, (int)groups, st); break;
    default: launch_read<256, 8>(p, (int)groups, st); break;
  }
  return launch_check(who);
}
