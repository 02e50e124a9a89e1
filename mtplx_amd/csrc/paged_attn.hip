// Causal attention of new tokens over the paged KV cache, from one decoded row
// per request to whole prompts, mixed as they come.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= position of i,
//
// in one pass over the keys with the running maximum m and sum l of each row:
// a block of scores s gives p = 2^(s log2e scale - m), l += sum p, o += p v.
// m moves only when a block's maximum passes it by 8 (then o and l are scaled
// by 2^(old - new)): p stays below 2^8 and fp32 carries the rest (sums are finite
// while the largest |v| times the keys stays below 2^120), and most blocks cost
// no pass over o.
//
// The query rows of the heads that share a kv head are one list per request
// (row r = token r / rep, head r % rep), cut into tiles of 32, 128 or 256 rows
// wherever that falls, so K and V are read once for all of them and 512 tokens
// of five heads are ten tiles (whole tokens, 51 a tile, took eleven: a chunk of
// 512 at 16k 202 us, now 184). S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16: a lane
// holds one query row's scores, so the maximum and sum over keys are its own
// registers' and one exchange with lane + 32, and P^T is already laid out as
// the second product's operand.
//
// 8-bit pages: integers are exact in bf16, so K and V enter the products as
// they are stored and their rows' scales multiply scores and weights in fp32.
// P is rounded to bf16 (as the values of V are), l sums it before that.
//
// Work is dealt by keys: every (request, kv head, row tile) is as long as the
// keys it sees plus a fixed cost, and workgroup g takes the g-th equal share
// of the whole line, whatever the lengths are. A tile that falls to more than
// one workgroup leaves one partial (o, m, l) per piece, at most two per
// workgroup, and attn_join adds them in the line's order. The split depends on
// lengths alone, so results do not depend on timing.
//
// What bounds it, on an MI355X (5.17 TB/s a large copy, 1350 TFLOP/s a large
// bf16 product), 40 query heads over 8 kv heads of 128:
//   sixteen requests' four verify rows up to 32k, 8 bits: 122 us, the pages at
//     the rate of the copy;
//   a chunk of 512 over 16k: 190 us, 890 TFLOP/s of what the mask leaves; whole
//     prompts of 4096: 519 us, 730 (diagonal blocks are computed whole). The
//     softmax's instructions (an exponential, a product, a maximum, a sum and
//     half a conversion a score) take as many cycles of a SIMD as the MFMAs,
//     and the two waves of a SIMD take them in turn: in the chunk the matrix
//     pipes are busy 50% of the CUs' busy cycles, vector issue 49%;
//   head dim 64: the chunk 117 us, the verify rows 76; head dim 256: 1377 (16
//     bits: registers spill inside the step) and 531 (8 bits), the verify rows 230;
//   one token over 4k: 17.7 us, of which the two launches' kernels are 12 and 5.
#include "paged.hpp"
#include "qmv_common.hpp"

#include <float.h>

#include <type_traits>

namespace mtp {

constexpr int kPT = 256;   // threads: four waves

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

struct PAttn {
  const uint16_t* q;
  uint16_t* out;
  const unsigned char* k_pages;
  const unsigned char* v_pages;
  const float* k_scales;
  const float* v_scales;
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* row_off;
  int32_t* status;
  float* part_o;    // [2 G][rows of a tile][D]
  float* part_ml;   // [2 G][rows of a tile][2]
  int4* begun;      // [G]: the tile that workgroup g began and others finish
  int T, B, width, Hq, Hkv, rep, bpp, num_pages;
  uint32_t rep_inv;   // row / rep = row * rep_inv >> 16 for rows below 2048
  int P;            // tokens that the rows of a tile may belong to
  int G;            // most workgroups
  int min_share;    // least keys of a workgroup's share
  int rt_log2;      // rows of a tile
  int step;         // shares are whole numbers of steps
  int tile_cost;
  float scale_log2;
  long long q_token, q_head, out_token, out_head;
};

// Token and head (of those that share a kv head) of a row of a tile's list.
__device__ __forceinline__ int row_token(const PAttn& p, int r) { return (int)(((uint32_t)r * p.rep_inv) >> 16); }

// -- the line of work -------------------------------------------------------------


struct Req {
  int lo, n;          // packed rows
  long long start;    // position of the first
  long long base;     // line position where its first head begins
  long long head;     // line length of one head
};

// Line length of a request's first t row tiles (one head).
__device__ __forceinline__ long long tiles_len(long long q0, int n, int P, long long t) {
  // sum over tiles x < t of q0 + min((x + 1) P, n): a tile's last row sees at
  // most that many keys (P: tokens that a tile's rows may belong to)
  const long long full = n / P;
  const long long f = t < full ? t : full;
  return t * q0 + P * (f * (f + 1) / 2) + (t - f) * n;
}
// (A tile's own cost, Q in and O out, counts as tile_cost keys.)
__device__ __forceinline__ long long clamp_start(const PAttn& p, long long s) {
  const long long cap = (long long)p.width * p.bpp * kBlk;
  return (s < 0 ? 0 : s > cap ? cap : s) + p.tile_cost;
}
// Row tiles of n tokens.
__device__ __forceinline__ int tile_count(const PAttn& p, int n) {
  return (int)(((long long)n * p.rep + (1 << p.rt_log2) - 1) >> p.rt_log2);
}
__device__ __forceinline__ long long head_len(const PAttn& p, long long start, int n) {
  return tiles_len(clamp_start(p, start), n, p.P, tile_count(p, n));
}

__device__ __forceinline__ long long shfl64(long long v, int src) { return __shfl(v, src, 64); }
__device__ __forceinline__ long long uniform64(long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (long long)((unsigned long long)hi << 32 | lo);
}

// a / b for a quotient below 2^31 (and a, b below 2^52), by an fp64 reciprocal
// with one Newton step (within one of it, then put right) instead of the integer
// division's long sequence.
__device__ __forceinline__ int div_small(long long a, long long b) {
  const double d = (double)b;
  double r = __builtin_amdgcn_rcp(d);
  r = fma(fma(-d, r, 1.0), r, r);
  int q = (int)((double)a * r);
  if ((long long)q * b > a) --q;
  if ((long long)(q + 1) * b <= a) ++q;
  return q;
}

// A lane's request of the line (64 requests at a time), its rows and length.
struct LaneReq {
  ReqRows rows;
  long long start, len;   // len: one head
};
__device__ __forceinline__ LaneReq lane_req(const PAttn& p, int b) {
  LaneReq r = {{0, 0}, 0, 0};
  if (b < p.B) {
    r.rows = req_rows(p.row_off, b, p.B, p.T);
    r.start = p.q_start[b];
    r.len = head_len(p, r.start, r.rows.n);
  }
  return r;
}
__device__ __forceinline__ long long scan64(long long v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const long long t = __shfl_up(v, off, 64);
    if (lane >= off) v += t;
  }
  return v;
}

// The line as a wave sees it: its total length W, cut into G shares of S.
struct Line {
  long long W, S;
  int G;
  __device__ __forceinline__ Line(const PAttn& p, int lane) {
    W = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) W += p.Hkv * lane_req(p, b0 + lane).len;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) W += __shfl_xor(W, off, 64);
    W = uniform64(W);
    // Equal shares, a whole number of steps each, no shorter than min_share.
    const long long s = W > 0 ? (W - 1) / p.G + 1 : 0;
    S = s > p.min_share ? (s + p.step - 1) & -(long long)p.step : p.min_share;
    G = W > 0 ? div_small(W - 1, S) + 1 : 0;
  }
  __device__ __forceinline__ long long lo(int g) const { return g * S; }
  __device__ __forceinline__ long long hi(int g) const { return g + 1 < G ? (g + 1) * S : W; }
  __device__ __forceinline__ int owner(long long x) const { return div_small(x, S); }
  // The request that holds line position x.
  __device__ __forceinline__ int find(const PAttn& p, int lane, long long x, Req& r) const {
    long long carry = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const LaneReq q = lane_req(p, b0 + lane);
      const long long end = scan64(p.Hkv * q.len, lane);
      const unsigned long long m = __ballot(q.len > 0 && x < carry + end);   // the first whose end lies behind x
      if (m) {
        const int src = __ffsll((long long)m) - 1;
        r.lo = __builtin_amdgcn_readfirstlane(__shfl(q.rows.lo, src, 64));
        r.n = __builtin_amdgcn_readfirstlane(__shfl(q.rows.n, src, 64));
        r.start = uniform64(shfl64(q.start, src));
        r.head = uniform64(shfl64(q.len, src));
        r.base = uniform64(carry + shfl64(end, src)) - p.Hkv * r.head;
        return __builtin_amdgcn_readfirstlane(b0 + src);
      }
      carry += shfl64(end, 63);
    }
    return -1;   // (not reached: x < W)
  }
};

// One row tile of one head: where it lies on the line and what it is. Tiles are
// whole whatever the heads of a kv head: a token's rows may lie in two of them.
struct Tile {
  long long begin, len;   // line
  int h, t;               // kv head, row tile
  int tok, off, rows;     // its first row: token of the request, head of that token; its rows
  long long pos;          // position of its first token
  int nk;                 // keys it sees: [0, nk)
};
// All but begin and h, from t.
__device__ __forceinline__ void set_tile(const PAttn& p, const Req& r, Tile& u) {
  const int first = u.t << p.rt_log2;   // (rows of a call: below 2^31)
  const int left = r.n * p.rep - first;
  u.rows = left >> p.rt_log2 ? 1 << p.rt_log2 : left;
  u.tok = (int)((uint32_t)first / (uint32_t)p.rep);
  u.off = first - u.tok * p.rep;
  const long long cost = (long long)(u.t + 1) * p.P;
  u.len = clamp_start(p, r.start) + (cost < r.n ? cost : r.n);
  u.pos = r.start + u.tok;
  const long long cap = (long long)p.width * p.bpp * kBlk;
  const long long e = u.pos + row_token(p, u.off + u.rows - 1) + 1;
  u.nk = (int)(e < 0 ? 0 : e > cap ? cap : e);
}
__device__ __forceinline__ Tile tile_at(const PAttn& p, const Req& r, long long x) {
  Tile u;
  const long long y = x - r.base;
  u.h = div_small(y, r.head);
  const long long z = y - u.h * r.head;
  const long long q0 = clamp_start(p, r.start);
  int a = 0, b = tile_count(p, r.n) - 1;   // the last tile that begins at or before z
  while (a < b) {
    const int m = (a + b + 1) >> 1;
    if (tiles_len(q0, r.n, p.P, m) <= z) a = m; else b = m - 1;
  }
  u.t = a;
  u.begin = r.base + u.h * r.head + tiles_len(q0, r.n, p.P, a);
  set_tile(p, r, u);
  return u;
}

// The tile after u on the line, in the same request.
__device__ __forceinline__ void next_tile(const PAttn& p, const Req& r, Tile& u) {
  u.begin += u.len;
  ++u.t;
  if (u.t == tile_count(p, r.n)) {
    u.t = 0;
    ++u.h;
  }
  set_tile(p, r, u);
}

// Keys [0, key_at(x)) of the tile lie before offset x of its line: whole steps
// of `step` keys.
__device__ __forceinline__ int key_at(const Tile& u, long long x, int step) {
  if (x >= u.len) return u.nk;
  const long long k = x / step * step;
  return k < u.nk ? (int)k : u.nk;
}

// -- one block of 32 keys ---------------------------------------------------------

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum with lane + 32's.
__device__ __forceinline__ float max_halves(float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); }

// A lane's query row (lane % 32 of the wave's 32): operands, running output,
// maximum and sum.
template <int D>
struct RowState {
  bf16x8 q[D / 16];
  f32x16 o[D / 32];
  float m, l;
  int bound;   // last key that the row sees; -1: none, or no row here
};

// Keys (bit k: key k of the block) of a 16-bit V block with a NaN or an
// infinity in any element; the same in every lane.
template <int D, class VO>
__device__ __forceinline__ uint32_t odd_keys(VO vop, int h2) {
  // An exponent of all ones plus one carries into the sign's place, half by half.
  u32x4 a0 = {}, a1 = {};
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    a0 |= (vop(t, 0) & 0x7f807f80u) + 0x00800080u;
    a1 |= (vop(t, 1) & 0x7f807f80u) + 0x00800080u;
  }
  const u32x4 a = a0 | a1;
  if (!__any((a.x | a.y | a.z | a.w) & 0x80008000u)) return 0;
  auto two = [&](uint32_t w, int i) {
    return (w >> 15 & 1u) << v_slot_key(h2, 2 * i) | (w >> 31) << v_slot_key(h2, 2 * i + 1);
  };
  uint32_t keys = two(a0.x, 0) | two(a0.y, 1) | two(a0.z, 2) | two(a0.w, 3) |
                  (two(a1.x, 0) | two(a1.y, 1) | two(a1.z, 2) | two(a1.w, 3)) << 16;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) keys |= __shfl_xor((int)keys, off, 64);
  return __builtin_amdgcn_readfirstlane((int)keys);
}

// A step's KB blocks of 32 keys from kt on go through three phases, each with
// its operands from where the caller keeps them (as 16 bytes of bf16).

// S^T = K Q^T. kop(j, i): operand i of block j.
template <int D, int KB, class KO>
__device__ __forceinline__ void scores(const RowState<D>& s, f32x16 (&st)[KB], KO kop) {
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    st[j] = f32x16{};
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      st[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kop(j, i)), s.q[i], st[j], 0, 0, 0);
  }
}

// Scores to weights (the second product's operand), the running maximum and
// sum. ks(j, r), vs(j, r): scales of the lane's key of score register r (8
// bits), ks already times scale_log2. MASK: the row sees keys up to its bound,
// of block j none at or past end[j].
template <int D, int BITS, int KB, bool MASK, class KS, class VS>
__device__ __forceinline__ void soften(RowState<D>& s, f32x16 (&st)[KB], u32x4 (&w)[KB][2], int kt,
                                       const int (&end)[KB], int h2, float scale_log2, KS ks, VS vs) {
  // 16 bits without a mask: the maximum is taken before the scale (positive),
  // and scale and maximum go into one FMA.
  constexpr bool RAW = BITS == 16 && !MASK;
  const int bound = s.bound - kt;
  auto hidden = [&](int j, int r) {   // (one comparison of a constant with what block j's registers share)
    const int last = (bound < end[j] - 1 - kt ? bound : end[j] - 1 - kt) - 32 * j - 4 * h2;
    return 8 * (r >> 2) + (r & 3) > last;
  };
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < KB; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = st[j][r];
      if (!RAW) x *= BITS == 8 ? ks(j, r) : scale_log2;
      if (MASK && hidden(j, r)) x = -INFINITY;
      st[j][r] = x;
      top = __builtin_elementwise_maximum(top, x);   // (no quieting of each x; a NaN makes its row NaN)
    }
  top = max_halves(top);
  if (RAW) top *= scale_log2;
  // A row that sees a key (of a block the first, then) has a finite maximum, so
  // it ends with l = 0 and m finite where all its scores are -infinity: NaN.
  bool sees = !MASK;
#pragma unroll
  for (int j = 0; j < KB; ++j) sees = sees || (kt + 32 * j <= s.bound && kt + 32 * j < end[j]);
  if (sees) top = fmaxf(top, -FLT_MAX);
  if (__any(top > s.m + 8.f)) {
    // Only the rows that passed: the others' bits do not turn on their neighbours.
    const float m_new = top > s.m + 8.f ? top : s.m;
    const float corr = s.m == -INFINITY ? 0.f : exp2_fast(s.m - m_new);
    s.m = m_new;
    s.l *= corr;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s.o[t][r] *= corr;
  }
  const float m = s.m == -INFINITY ? 0.f : s.m;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    uint32_t pk[8];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      auto weight = [&](int rr) {
        const float x = st[j][rr];
        return exp2_fast(RAW ? __fmaf_rn(x, scale_log2, -m) : x - m);
      };
      float a = weight(r), b = weight(r + 1);
      sum += a + b;
      if (BITS == 8) {
        const float va = vs(j, r), vb = vs(j, r + 1);
        a = MASK && hidden(j, r) ? 0.f : a * va;   // (a hidden key's scale may be NaN; of one that is seen it shows)
        b = MASK && hidden(j, r + 1) ? 0.f : b * vb;
      }
      pk[r / 2] = f2bf2(a, b);
    }
    w[j][0] = u32x4{pk[0], pk[1], pk[2], pk[3]};
    w[j][1] = u32x4{pk[4], pk[5], pk[6], pk[7]};
  }
  s.l += sum;
}

// O^T += V^T P^T of block j's weights w. vop(t, jj): its operands. MASK, 16
// bits: a hidden key's weight is 0, but 0 times a NaN or an infinity in its
// value is not: keys whose values are not all finite leave the product and are
// added one by one, to the rows that see them; at or past `end` there is
// nothing. (8-bit values are integers; their scale went into the weight.)
template <int D, int BITS, bool MASK, class VO>
__device__ __forceinline__ void add_values(RowState<D>& s, const u32x4 (&w)[2], int kt, int end, int h2, VO vop) {
  u32x4 keep0 = {}, keep1 = {};
  uint32_t odd = 0;
  if (MASK && BITS == 16) {
    const int n = end - kt;   // keys that exist
    const uint32_t have = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
    odd = odd_keys<D>(vop, h2) & have;
    const uint32_t in = have & ~odd;
    auto word = [&](int jj, int i) {
      return (in >> (16 * jj + v_slot_key(h2, 2 * i)) & 1 ? 0x0000ffffu : 0u) |
             (in >> (16 * jj + v_slot_key(h2, 2 * i + 1)) & 1 ? 0xffff0000u : 0u);
    };
    keep0 = u32x4{word(0, 0), word(0, 1), word(0, 2), word(0, 3)};
    keep1 = u32x4{word(1, 0), word(1, 1), word(1, 2), word(1, 3)};
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      u32x4 v = vop(t, jj);
      if (MASK && BITS == 16) v &= jj ? keep1 : keep0;
      s.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, w[jj]),
                                                       s.o[t], 0, 0, 0);
    }
  if (MASK && BITS == 16) {
    for (; odd; odd &= odd - 1) {
      const int key = __ffs((int)odd) - 1, r = key & 15;
      const int e = r < 8 ? (r & 3) : 4 + (r & 3);
      const uint32_t half = h2 != (r & 7) >> 2 ? 0u : e & 1 ? 0xffff0000u : 0x0000ffffu;
      const uint32_t low = key < 16 ? 0xffffffffu : 0u;
      const int word = e >> 1;
      const u32x4 only = {word == 0 ? half : 0u, word == 1 ? half : 0u, word == 2 ? half : 0u, word == 3 ? half : 0u};
      const u32x4 wn = (w[0] & low) | (w[1] & ~low);
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        const u32x4 v = ((vop(t, 0) & low) | (vop(t, 1) & ~low)) & only;
        const f32x16 add = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v),
                                                                   __builtin_bit_cast(bf16x8, wn), f32x16{}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) s.o[t][i] += kt + key <= s.bound ? add[i] : 0.f;
      }
    }
  }
}

// Where the blocks of a request's key range lie in the pool (block ordinals),
// 64 at a time: lane l keeps block `first` + l's, so the key loop looks nothing
// up in memory (a load there would wait for every tile in flight). Blocks
// without a page (bits of `gone`) are given ordinal 0: what is read there is
// never used.
struct BlockList {
  unsigned long long gone;
  int at, first;
  __device__ __forceinline__ void fill(const PAttn& p, int b, int h, int blk, int end, int lane) {
    first = blk;
    at = blk + lane < end ? (int)page_block(p.table, p.width, b, blk + lane, p.bpp, p.num_pages, p.Hkv, h, 1) : -1;
    if (p.status && blk + lane < end && at < 0) atomicOr(p.status, kStatusPage);
    gone = __ballot(at < 0);
    if (at < 0) at = 0;
  }
  __device__ __forceinline__ int get(int blk) const { return __builtin_amdgcn_readlane(at, blk - first); }
  __device__ __forceinline__ bool absent(int blk) const { return gone >> (blk - first) & 1; }
  // Leading blocks of the list that have a page.
  __device__ __forceinline__ int present() const { return gone ? __ffsll((long long)gone) - 1 : 64; }
};

// Rows row0 .. of a tile (row r of the list: token r / rep, head r % rep), 32 of
// a wave. A lane's operands lie all over its row, so the rows come whole, 16
// bytes a lane, and turn through LDS (RB bytes a row, the wave's own).
template <int D>
constexpr int row_bytes() { return D * 2 + 16; }   // (reads of 8 rows hit distinct banks)

template <int D>
struct RowLoads {
  u32x4 r[D / 16];
};
template <int D>
__device__ __forceinline__ void ask_rows(RowLoads<D>& q, const PAttn& p, const Req& rq, const Tile& u, int row0,
                                         int lane) {
  constexpr int LPR = D / 8;   // lanes of a row
  lane = fresh(lane);
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    const int r = row0 + j * (64 / LPR) + lane / LPR;
    int i = row_token(p, r + u.off), g = r + u.off - i * p.rep;
    if (r >= u.rows) i = g = 0;   // no row here: any
    const long long tok = (long long)rq.lo + u.tok + i;
    q.r[j] = *reinterpret_cast<const u32x4*>(p.q + tok * p.q_token + (long long)(u.h * p.rep + g) * p.q_head +
                                             lane % LPR * 8);
  }
}
template <int D>
__device__ __forceinline__ void take_rows(RowState<D>& s, const RowLoads<D>& q, const PAttn& p, const Tile& u, int row0,
                                          int lane, unsigned char* lds) {
  constexpr int LPR = D / 8, RB = row_bytes<D>();
  lane = fresh(lane);
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
    *reinterpret_cast<u32x4*>(lds + (j * (64 / LPR) + lane / LPR) * RB + lane % LPR * 16) = q.r[j];
  const int h2 = lane >> 5, r = row0 + (lane & 31);
  const int i = row_token(p, r + u.off);
  const bool valid = r < u.rows;
  const long long pos = u.pos + i;
  s.bound = !valid || pos < 0 ? -1 : pos < u.nk ? (int)pos : u.nk - 1;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    const u32x4 raw = *reinterpret_cast<const u32x4*>(lds + (lane & 31) * RB + D * h2 + 16 * j);
    s.q[j] = __builtin_bit_cast(bf16x8, valid ? raw : u32x4{0, 0, 0, 0});
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t) s.o[t] = f32x16{};
  s.m = -INFINITY;
  s.l = 0.f;
}

// Partials: float4 e of (32 rows, 32 d) block (row block, t) is row e % 32 and
// d = 4 (e / 32): the registers' own order, 1 KB a store.
template <int D>
__device__ __forceinline__ float4* part_block(const PAttn& p, size_t slot, int RT, int rb, int t) {
  return reinterpret_cast<float4*>(p.part_o) + ((slot * (RT / 32) + rb) * (D / 32) + t) * 256;
}

// The factor of a row's sums in its output: a row that saw no key is zeros.
__device__ __forceinline__ float row_factor(float m, float l) { return m == -INFINITY && l == 0.f ? 0.f : 1.f / l; }

// 16 bytes read once per launch (non-temporal, as ld_stream).
__device__ __forceinline__ u32x4 ld_nt(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// Four consecutive d of an output row.
__device__ __forceinline__ void store4(uint16_t* dst, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(f2bf2(a, b), f2bf2(c, d));
}

// Row r (from the first head of token `token`, packed, on) of kv head h.
__device__ __forceinline__ uint16_t* out_row(const PAttn& p, int token, int h, int r) {
  const int i = row_token(p, r), g = r - i * p.rep;
  return p.out + ((long long)token + i) * p.out_token + (long long)(h * p.rep + g) * p.out_head;
}

// What the join needs to know of the tile that workgroup g begins and others
// finish (at most one).
__device__ __forceinline__ void note_begun(const PAttn& p, const Line& line, const Req& rq, const Tile& u, int g) {
  const int last = line.owner(u.begin + u.len - 1);
  p.begun[g] = make_int4(u.rows | u.off << 16, (last < line.G ? last : line.G - 1) - g + 1, rq.lo + u.tok, u.h);
}

// Byte I of w, signed, as a float: one instruction (the compiler takes two, a
// bit field and a conversion).
template <int I>
__device__ __forceinline__ float byte_f32(uint32_t w) {
  float f;
  if constexpr (I == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
  if constexpr (I == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
  if constexpr (I == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
  if constexpr (I == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
  return f;
}

// Eight bytes of integers -> eight bf16 (exact).
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  return u32x4{f2bf2(byte_f32<0>(a), byte_f32<1>(a)), f2bf2(byte_f32<2>(a), byte_f32<3>(a)),
               f2bf2(byte_f32<0>(b), byte_f32<1>(b)), f2bf2(byte_f32<2>(b), byte_f32<3>(b))};
}

// -- chunks: row tiles of 32 NB rows a wave, K and V tiles shared through LDS ----

constexpr int kStepKeys = 64;

// Two waves of 32 rows on a SIMD; at D = 256 one (its accumulators and queries
// take 192 registers).
template <int D>
constexpr int chunk_waves() { return D == 256 ? 4 : 8; }

// Between two barriers a wave computes a step's products (PV of step n - 1, then
// QK of n) and a softmax, and the two waves of a SIMD (w and w + 4) do so in
// turn: the first four products(n), softmax(n), the others softmax(n - 1),
// products(n), so one's matrix instructions run beside the other's exponentials.
//
// With step n's products a wave also stores its share of K and V of step n + 1,
// loaded a step before, and loads those of n + 2: V(n) lies there a step before
// its product, whose first operands are read ahead of the barrier. (Loads
// straight into LDS stall the wave that issues them, 600 to 1000 cycles of a
// step.)
template <int D, int BITS>
__global__ __launch_bounds__(64 * chunk_waves<D>()) void attn_chunk_kernel(PAttn p) {
  constexpr int NW = chunk_waves<D>(), NT = 64 * NW;
  constexpr int RT = NW * 32;
  constexpr int BE = kBlk * D;                      // elements of a block
  constexpr int CB = BE * (BITS / 8) / 16;          // 16-byte chunks of a block
  constexpr int LD = 2 * CB / NT > 0 ? 2 * CB / NT : 1;   // a thread's, of a step's two blocks
  // K of a step lives for two phases and is written in the two before; V lives
  // for four (at D = 256, where no wave runs half a step behind, for two).
  constexpr int KR = 2, VR = D == 256 ? 2 : 3;
  __shared__ __attribute__((aligned(16))) unsigned char lds[(KR + VR) * 4 * BE];   // K slots, then V's
  static_assert(NW * 32 * row_bytes<D>() <= (KR + VR) * 4 * BE, "a wave's rows turn in the slots' place");
  __shared__ __attribute__((aligned(16))) float ksc[4][kStepKeys], vsc[4][kStepKeys];   // (of step n - 1 to n + 1)
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Line line(p, lane);
  if (tid == 0 && (int)blockIdx.x >= line.G) p.begun[blockIdx.x] = make_int4(0, 0, 0, 0);
  // Neighbours on the line share a head's keys: they go to one XCD (workgroups
  // are dealt to the eight in turn), whose L2 then serves them.
  const int per = cdiv(line.G, 8);
  const int g = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if ((int)blockIdx.x >> 3 >= per || g >= line.G) return;
  if (tid == 0) p.begun[g] = make_int4(0, 0, 0, 0);
  const long long lo = line.lo(g), hi = line.hi(g);
  const int turn = NW == 8 && wave >= 4 ? 1 : 0;
  const uint32_t klds = lds_addr(lds), vlds = klds + KR * 4 * BE;
  Req rq;
  int b = line.find(p, lane, lo, rq);
  Tile u = tile_at(p, rq, lo);
  for (long long x = lo; x < hi;) {
    if (x >= rq.base + p.Hkv * rq.head) {
      b = line.find(p, lane, x, rq);
      u = tile_at(p, rq, x);
    } else if (x >= u.begin + u.len) {
      next_tile(p, rq, u);
    }
    const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
    const int ka = key_at(u, x - u.begin, kStepKeys), kb = key_at(u, end - u.begin, kStepKeys);
    const bool starts = x == u.begin, ends = end == u.begin + u.len;
    x = end;
    if (starts && !ends && tid == 0) note_begun(p, line, rq, u, g);
    const int row0 = wave * 32;
    const int rows = u.rows;
    RowLoads<D> ql;
    ask_rows<D>(ql, p, rq, u, row0, lane);
    // Bounds of the wave's rows: steps behind wmax are skipped, steps up to
    // wmin need no mask (rows past the list are computed on zeros, and dropped).
    const int last = (row0 + 32 < rows ? row0 + 32 : rows) - 1;
    long long wmin = u.pos + row_token(p, row0 + u.off);
    const long long wmax = row0 < rows ? u.pos + row_token(p, last + u.off) : -1;
    if (wmin > u.nk - 1) wmin = u.nk - 1;

    BlockList blocks;
    blocks.fill(p, b, u.h, ka >> 5, (kb + 31) >> 5, lane);
    const int nstep = (kb - ka + kStepKeys - 1) / kStepKeys;
    // Steps [0, nfull) hide no key from any of the wave's rows and have all
    // their pages; [nfull, nlive) hide some; the rest hides all.
    int nfull = 0, nlive = 0;
    if (wmax >= ka) nlive = wmax >= kb ? nstep : (int)((wmax - ka) / kStepKeys) + 1;
    if (nlive > 0 && wmin + 1 - ka >= kStepKeys) nfull = (int)((wmin + 1 - ka) / kStepKeys);
    if (nfull > nlive) nfull = nlive;
    auto cut = [&](int st) {   // the list begins at step st: its steps before the first absent block
      const int lead = st + (blocks.present() >> 1);
      if (lead < nfull && lead < st + 32) nfull = lead;
    };
    cut(0);
    // A list that step st ends is replaced while steps from `from` on still use
    // it: lists overlap.
    const int blk0 = ka >> 5, blk1 = (kb + 31) >> 5;
    auto cover = [&](int from, int st) {
      if (blk0 + 2 * st + 2 > blocks.first + 64) {
        blocks.fill(p, b, u.h, blk0 + 2 * from, blk1, lane);
        cut(from);
      }
    };
    u32x4 kr[LD], vr[LD];   // a step's K and V on their way to LDS
    float kscale = 0.f, vscale = 0.f;
    // The thread's share of K and V of step st (past the last: the last one's
    // again, never used).
    auto load = [&](int st, bool isv) {
      const int blk = blk0 + 2 * (st < nstep ? st : nstep - 1);
      const int a0 = blocks.get(blk), a1 = blocks.get(blk + 1);
      const unsigned char* pool = isv ? p.v_pages : p.k_pages;
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int c = i * NT + wave * 64;   // the wave's first chunk: uniform, 64 chunks lie in one block
        if (2 * CB % NT && c >= 2 * CB) break;
        const bool second = CB % NT ? c >= CB : i * NT >= CB;
        const unsigned char* src = pool + (size_t)(second ? a1 : a0) * (CB * 16) + (second ? c - CB : c) * 16;
        const u32x4 r = *reinterpret_cast<const u32x4*>(src + (uint32_t)(lane * 16));
        if (isv) vr[i] = r; else kr[i] = r;
      }
      if (BITS == 8 && !isv && tid < kStepKeys) {
        const size_t o = (size_t)(tid >= 32 ? a1 : a0) * kBlk + (tid & 31);
        kscale = p.k_scales[o];
        vscale = p.v_scales[o];
      }
    };
    auto load_next = [&](int n) {   // with step n's products
      load(n + 2, false);
      load(n + VR - 1, true);
    };
    auto put = [&](uint32_t dst, const u32x4 (&r)[LD]) {   // LDS addresses
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int c = i * NT + wave * 64;
        if (2 * CB % NT && c >= 2 * CB) break;
        lds_u32x4* d = reinterpret_cast<lds_u32x4*>(dst + lane * 16 + c * (BITS == 16 ? 16 : 32));
        if constexpr (BITS == 16) {
          d[0] = r[i];
        } else {   // 64 chunks of 16 integers to two operands of 64 x 8
          d[0] = widen8(r[i].x, r[i].y);
          d[64] = widen8(r[i].z, r[i].w);
        }
      }
    };
    // Ring slots: K of steps n and n + 1; V of n - 1, n and (of three) n + 1.
    int k0 = 0, k1 = 1, v0 = VR - 1, v1 = 0, v2 = 1;
    auto turn_ring = [&] {
      const int k = k0, v = v0;
      k0 = k1;
      k1 = k;
      v0 = v1;
      v1 = VR == 3 ? v2 : v;
      v2 = v;
    };
    auto store_k = [&](int n) {   // of step n (slot k1 when n is the next step)
      put(klds + k1 * (4 * BE), kr);
      if (BITS == 8 && tid < kStepKeys) {
        ksc[n & 3][tid] = kscale * p.scale_log2;
        vsc[n & 3][tid] = vscale;
      }
    };
    auto store_v = [&] { put(vlds + (VR == 3 ? v2 : v1) * (4 * BE), vr); };   // of step n + 1 (two slots: n)
    if (nstep > 0) {   // step 0 in LDS (its V on the way, of two slots), step 1 on its way
      load(0, false);
      load(0, true);
    }
    unsigned char* const mine = lds + wave * (32 * row_bytes<D>());   // (of no step: between pieces)
    RowState<D> s;
    take_rows<D>(s, ql, p, u, row0, lane, mine);
    f32x16 st[2];
    u32x4 w[2][2];
    u32x4 op[2][D / 16];
    // Operands from a ring slot: one address, offsets in the instructions.
    auto operands = [&](uint32_t lds, int ring) {
      uint32_t a = lds + ring * (4 * BE) + lane * 16;
      asm("" : "+v"(a));
      return reinterpret_cast<const lds_u32x4*>(a);
    };
    auto ask = [&](u32x4 (&to)[D / 16], const lds_u32x4* from, int j) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) to[i] = from[(j * (D / 16) + i) * 64];
      __builtin_amdgcn_sched_barrier(0);
    };
    auto keys = [&] {
      const lds_u32x4* k = operands(klds, k0);
      scores<D, 2>(s, st, [&](int j, int i) { return k[(j * (D / 16) + i) * 64]; });
    };
    auto ends2 = [&](int n, int j) { return blocks.absent(blk0 + 2 * n + j) ? 0 : u.nk; };
    auto values = [&](int n) {   // of step n, masked; slot v0 when n is the last step
      const lds_u32x4* v = operands(vlds, v0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        add_values<D, BITS, true>(s, w[j], ka + n * kStepKeys + 32 * j, ends2(n, j), h2,
                                  [&](int t, int jj) { return v[(j * (D / 16) + 2 * t + jj) * 64]; });
    };
    // Both products of step n, no key hidden: each eight operands are asked for
    // eight matrix instructions ahead (left alone, the compiler reads one, waits
    // for it and multiplies); op[0] is in hand.
    auto products = [&](int n) {
      const lds_u32x4* v = operands(vlds, v0);
      const lds_u32x4* k = operands(klds, k0);
      auto add = [&](const u32x4 (&from)[D / 16], int j) {
        add_values<D, BITS, false>(s, w[j], 0, 0, h2, [&](int t, int jj) { return from[2 * t + jj]; });
        __builtin_amdgcn_sched_barrier(0);
      };
      auto score = [&](const u32x4 (&from)[D / 16], int j) {
        f32x16 one[1];
        scores<D, 1>(s, one, [&](int, int i) { return from[i]; });
        st[j] = one[0];
        __builtin_amdgcn_sched_barrier(0);
      };
      if (VR == 2) ask(op[0], v, 0);
      ask(op[1], v, 1);
      add(op[0], 0);
      ask(op[0], k, 0);
      store_k(n + 1);
      add(op[1], 1);
      ask(op[1], k, 1);
      store_v();
      score(op[0], 0);
      load_next(n);
      score(op[1], 1);
    };
    // Scores to weights. (They are not to be touched before the barrier that ends
    // the products phase: moved ahead of it, the softmax would keep the other
    // waves waiting.)
    auto weights = [&](int n, auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" : "+v"(st[0]), "+v"(st[1]));
      const float* kss = &ksc[n & 3][4 * h2];
      const float* vss = &vsc[n & 3][4 * h2];
      const int end[2] = {MASK ? ends2(n, 0) : 0, MASK ? ends2(n, 1) : 0};
      soften<D, BITS, 2, MASK>(
          s, st, w, ka + n * kStepKeys, end, h2, p.scale_log2,
          [&](int j, int r) { return kss[32 * j + 8 * (r >> 2) + (r & 3)]; },
          [&](int j, int r) { return vss[32 * j + 8 * (r >> 2) + (r & 3)]; });
    };
    auto look_ahead = [&] {   // the next products' first operands: V of the step just softened
      if (VR == 3) ask(op[0], operands(vlds, v0), 0);
    };
    constexpr std::true_type yes;
    constexpr std::false_type no;
    lds_barrier();   // every wave has its rows
    if (nstep > 0) {
      put(klds, kr);
      if (BITS == 8 && tid < kStepKeys) {
        ksc[0][tid] = kscale * p.scale_log2;
        vsc[0][tid] = vscale;
      }
      load(1, false);
      if (VR == 3) {
        put(vlds, vr);
        load(1, true);
      }
      lds_barrier();
      auto stage = [&](int n) {   // what goes with step n's products
        store_k(n + 1);
        store_v();
        cover(n > 0 ? n - 1 : 0, n + 2);
        load_next(n);
      };
      auto between = [&] {   // products and softmax
        if (turn) lds_barrier();
      };
      auto after = [&] {
        turn_ring();
        if (!turn) lds_barrier();
      };
      // Full steps, then steps that may hide keys, then (for the other waves)
      // staging alone; straight lines between, so the accumulators stay where
      // they are.
      int n = 0;
      if (nfull > 0) {
        keys();
        stage(0);
        between();
        weights(0, no);
        after();
        look_ahead();
        for (n = 1; n < nfull; ++n) {
          cover(n - 1, n + 2);
          products(n);
          between();
          weights(n, no);
          after();
          look_ahead();
        }
      } else if (nlive > 0) {
        keys();
        stage(0);
        between();
        weights(0, yes);
        after();
        n = 1;
      }
      for (; n < nlive; ++n) {
        values(n - 1);
        keys();
        stage(n);
        between();
        weights(n, yes);
        after();
      }
      if (nlive > 0) values(nlive - 1);
      for (; n < nstep; ++n) {
        stage(n);
        between();
        after();
      }
    }
    // Out: the whole tile's rows (turned through LDS, as they came), or this
    // piece's partial (without keys: m = -infinity, l = 0, and its o is not read).
    const float l = s.l + __shfl_xor(s.l, 32, 64);
    lds_barrier();   // every wave is done with the slots
    const int ln = fresh(lane);
    if (starts && ends) {
      constexpr int LPR = D / 8, RB = row_bytes<D>();
      const float inv = row_factor(s.m, l);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          store4(reinterpret_cast<uint16_t*>(mine + (ln & 31) * RB) + 32 * t + 8 * j + 4 * (ln >> 5), s.o[t][4 * j] * inv,
                 s.o[t][4 * j + 1] * inv, s.o[t][4 * j + 2] * inv, s.o[t][4 * j + 3] * inv);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int r = j * (64 / LPR) + ln / LPR;
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * RB + ln % LPR * 16);
        if (row0 + r < rows)
          *reinterpret_cast<u32x4*>(out_row(p, rq.lo + u.tok, u.h, row0 + r + u.off) + ln % LPR * 8) = v;
      }
    } else if (row0 < rows) {
      const size_t slot = 2 * (size_t)g + (starts ? 1 : 0);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          part_block<D>(p, slot, RT, wave, t)[j * 64 + ln] =
              make_float4(s.o[t][4 * j], s.o[t][4 * j + 1], s.o[t][4 * j + 2], s.o[t][4 * j + 3]);
      if (ln < 32) {
        float* ml = p.part_ml + (slot * RT + row0 + ln) * 2;
        ml[0] = s.m;
        ml[1] = l;
      }
    }
  }
}

// -- few rows: one tile of 32 rows, the four waves share a piece by keys ---------

// Blocks go straight from the pages into a wave's registers, the next one asked
// for as soon as this one's operands are used up. Two workgroups a CU where
// their registers allow (D < 256): sixteen requests' verify rows at 8 bits take
// 122 us, with one 149.
template <int D, int BITS>
__global__ __launch_bounds__(kPT, D == 256 ? 1 : 2) void attn_few_kernel(PAttn p) {
  constexpr int RT = 32;
  constexpr int BE = kBlk * D;
  constexpr int LD = D / 16 * (BITS / 8) / 2;   // 16-byte loads of a lane per block
  constexpr int OS = D + 4;                     // padded row: lanes of one store hit distinct banks
  __shared__ __attribute__((aligned(16))) float s_o[4][32 * OS];
  __shared__ float s_m[4][32], s_l[4][32];
  const int tid = threadIdx.x, lane = tid & 63, c32 = lane & 31, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Line line(p, lane);
  const int g = blockIdx.x;
  if (tid == 0) p.begun[g] = make_int4(0, 0, 0, 0);
  if (g >= line.G) return;
  const long long lo = line.lo(g), hi = line.hi(g);
  Req rq;
  int b = line.find(p, lane, lo, rq);
  Tile u = tile_at(p, rq, lo);
  for (long long x = lo; x < hi;) {
    if (x >= rq.base + p.Hkv * rq.head) {
      b = line.find(p, lane, x, rq);
      u = tile_at(p, rq, x);
    } else if (x >= u.begin + u.len) {
      next_tile(p, rq, u);
    }
    const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
    const int ka = key_at(u, x - u.begin, kBlk), kb = key_at(u, end - u.begin, kBlk);
    const bool starts = x == u.begin, ends = end == u.begin + u.len;
    x = end;
    if (starts && !ends && tid == 0) note_begun(p, line, rq, u, g);
    const int rows = u.rows;
    RowLoads<D> q;
    ask_rows<D>(q, p, rq, u, 0, lane);
    const long long wmin = u.pos < u.nk - 1 ? u.pos : u.nk - 1;   // blocks up to it hide no key
    const int nblk = (kb - ka + kBlk - 1) / kBlk;
    const int b0 = (ka >> 5) + nblk * wave / 4, b1 = (ka >> 5) + nblk * (wave + 1) / 4;   // the wave's blocks
    BlockList blocks;
    if (b0 < b1) blocks.fill(p, b, u.h, b0, b1, lane);
    u32x4 kr[LD], vr[LD];
    float sc = 0.f;   // 8 bits: lane l's key's scale, of K (l < 32) and of V
    auto load = [&](int blk) {
      const size_t o = (size_t)blocks.get(blk < b1 ? blk : b1 - 1) * BE;   // (past the last: the last again, never used)
      const unsigned char* k = p.k_pages + o * (BITS / 8);
      const unsigned char* v = p.v_pages + o * (BITS / 8);
#pragma unroll
      for (int i = 0; i < LD; ++i) kr[i] = ld_nt(k + (uint32_t)(i * 1024 + lane * 16));
#pragma unroll
      for (int i = 0; i < LD; ++i) vr[i] = ld_nt(v + (uint32_t)(i * 1024 + lane * 16));
      if constexpr (BITS == 8) sc = (h2 ? p.v_scales : p.k_scales)[o / D + c32];
    };
    if (b0 < b1) load(b0);
    RowState<D> s;
    __syncthreads();   // the previous piece's reads of s_o are done
    take_rows<D>(s, q, p, u, 0, lane, reinterpret_cast<unsigned char*>(s_o[wave]));
    float* const scales = s_o[wave];   // 8 bits: a block's scales, on their way to the lanes that need them
    auto block = [&](int blk, auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      const int kt = 32 * blk;
      if constexpr (BITS == 8) scales[lane] = h2 ? sc : sc * p.scale_log2;
      auto scale = [&](int r) { return scales[8 * (r >> 2) + 4 * h2 + (r & 3)]; };
      f32x16 st[1];
      u32x4 w[1][2];
      const int end1[1] = {u.nk};
      scores<D, 1>(s, st, [&](int, int i) {
        if constexpr (BITS == 16) return kr[i];
        else return (i & 1) ? widen8(kr[i >> 1].z, kr[i >> 1].w) : widen8(kr[i >> 1].x, kr[i >> 1].y);
      });
      soften<D, BITS, 1, MASK>(
          s, st, w, kt, end1, h2, p.scale_log2, [&](int, int r) { return scale(r); },
          [&](int, int r) { return scale(r + 16); });
      if (BITS == 8) __builtin_amdgcn_sched_barrier(0);   // (V's integers are not widened before their turn)
      add_values<D, BITS, MASK>(s, w[0], kt, u.nk, h2, [&](int t, int jj) {
        if constexpr (BITS == 16) return vr[2 * t + jj];
        else return jj ? widen8(vr[t].z, vr[t].w) : widen8(vr[t].x, vr[t].y);
      });
    };
    auto next = [&](int blk) {   // the block after blk, in its place
      if (blk + 1 >= blocks.first + 64 && blk + 1 < b1) blocks.fill(p, b, u.h, blk + 1, b1, lane);
      load(blk + 1);
    };
    // Blocks [b0, bf) hide no key and have their pages.
    int bf = wmin + 1 >= 0 ? (int)((wmin + 1) >> 5) : 0;
    if (bf > b1) bf = b1;
    int blk = b0;
    while (blk < b1) {
      // As far as this list knows.
      int to = blocks.first + blocks.present();
      if (to > bf) to = bf;
#pragma unroll 1
      for (; blk < to; ++blk) {
        block(blk, std::false_type());
        next(blk);
        to = blocks.first + blocks.present() < bf ? blocks.first + blocks.present() : bf;
      }
      if (blk >= b1) break;
      if (!blocks.absent(blk)) block(blk, std::true_type());
      next(blk);
      ++blk;
    }
    // The waves' parts, in wave order.
    const float l = s.l + __shfl_xor(s.l, 32, 64);
    if (h2 == 0) {
      s_m[wave][c32] = s.m;
      s_l[wave][c32] = l;
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(&s_o[wave][c32 * OS + 32 * t + 8 * j + 4 * h2]) =
            make_float4(s.o[t][4 * j], s.o[t][4 * j + 1], s.o[t][4 * j + 2], s.o[t][4 * j + 3]);
    __syncthreads();
    const int slot = 2 * g + (starts ? 1 : 0);
    const bool whole = starts && ends;
    for (int e = tid; e < 8 * D; e += kPT) {   // (row e % 32, d = 4 (e / 32): the partials' order)
      const int r = e & 31, d = e >> 5 << 2;
      if (r >= rows) continue;
      float m = s_m[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) m = fmaxf(m, s_m[w][r]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float c = s_m[w][r] == -INFINITY ? 0.f : exp2_fast(s_m[w][r] - m);
        const float4 a = *reinterpret_cast<const float4*>(&s_o[w][r * OS + d]);
        v.x += a.x * c;
        v.y += a.y * c;
        v.z += a.z * c;
        v.w += a.w * c;
        ls += s_l[w][r] * c;
      }
      if (whole) {
        const float inv = row_factor(m, ls);
        store4(out_row(p, rq.lo + u.tok, u.h, r + u.off) + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        part_block<D>(p, slot, RT, 0, 0)[e] = v;
        if (d == 0) {
          float* ml = p.part_ml + ((size_t)slot * RT + r) * 2;
          ml[0] = m;
          ml[1] = ls;
        }
      }
    }
  }
}

// -- join: the tiles that fell to more than one workgroup ------------------------

// Workgroup (g, y): one (32 rows, 32 d) block of the tile that workgroup g began
// and others finished; a thread sums one float4 of it over the pieces, eight
// loads at a time, with the pieces' weights 2^(m - max) from LDS. Lanes without
// a row (a decode step's tile holds few) take a share of the pieces instead:
// with NR rows' lanes, lane r + NR s adds pieces s, s + 32 / NR, .. of row r.
template <int RT>
constexpr int join_round() { return RT == 32 ? 64 : 16; }   // pieces whose weights LDS holds

template <int D, int RT>
__global__ __launch_bounds__(kPT) void attn_join_kernel(PAttn p) {
  constexpr int kJoin = join_round<RT>();
  __shared__ float s_w[kJoin][32], s_m[32], s_l[32];
  __shared__ __attribute__((aligned(16))) uint16_t s_out[32][32 + 8];
  const int tid = threadIdx.x;
  const int g = blockIdx.x;
  const int4 tile = p.begun[g];   // rows (0: none) and first head, pieces, first token, kv head
  const int rows = tile.x & 0xffff, head0 = tile.x >> 16, np = tile.y;
  const int rb = blockIdx.y / (D / 32), t = blockIdx.y % (D / 32);
  const int r0 = 32 * rb;
  if (r0 >= rows) return;
  // Piece k's slot: the one that begins the tile is g's second.
  auto slot = [&](int k) { return (size_t)(2 * (g + k) + (k == 0 ? 1 : 0)); };
  int NR = 32;   // (chunks' tiles: always, so that the loop below is a plain one)
  while (RT == 32 && NR > 4 && rows - r0 <= NR / 2) NR >>= 1;
  const int SP = 32 / NR, row = tid & (NR - 1), share = (tid & 31) / NR;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int B8 = RT == 32 ? 8 : 4;   // pieces whose blocks are in flight together
  float4 a8[B8];
  auto ask = [&](int k) {   // (the last piece again past the last: never used)
#pragma unroll
    for (int i = 0; i < B8; ++i) {
      const int kk = k + SP * i + share;
      a8[i] = part_block<D>(p, slot(kk < np ? kk : np - 1), RT, rb, t)[(tid & ~31) + row];
    }
  };
  ask(0);
  if (tid < 32) {
    s_m[tid] = -INFINITY;
    s_l[tid] = 0.f;
  }
  for (int k0 = 0; k0 < np; k0 += kJoin) {
    const int n = np - k0 < kJoin ? np - k0 : kJoin;
    __syncthreads();
    const float m_old = s_m[row];
    __syncthreads();   // read before it is replaced
    // A row's weights by 8 lanes, eight pieces each at most.
    {
      const int rr = tid >> 3, x = tid & 7;
      const bool live = r0 + rr < rows;
      float2 a[kJoin / 8];
      const float old = s_m[rr];
      float m = old;
#pragma unroll
      for (int i = 0; i < kJoin / 8; ++i) {
        const int k = 8 * i + x;
        a[i] = make_float2(-INFINITY, 0.f);
        if (live && k < n) a[i] = *reinterpret_cast<const float2*>(p.part_ml + (slot(k0 + k) * RT + r0 + rr) * 2);
      }
#pragma unroll
      for (int i = 0; i < kJoin / 8; ++i) m = fmaxf(m, a[i].x);
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < kJoin / 8; ++i) {
        const float w = a[i].x == -INFINITY ? 0.f : exp2_fast(a[i].x - m);
        l += a[i].x == -INFINITY ? a[i].y : a[i].y * w;   // (no score: 0 or NaN)
        s_w[8 * i + x][rr] = w;
      }
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) l += __shfl_xor(l, off, 64);
      if (x == 0) {
        s_l[rr] = s_l[rr] * (old == -INFINITY ? 1.f : exp2_fast(old - m)) + l;
        s_m[rr] = m;
      }
    }
    __syncthreads();
    const float c = m_old == -INFINITY ? 0.f : exp2_fast(m_old - s_m[row]);
    v.x *= c;
    v.y *= c;
    v.z *= c;
    v.w *= c;
    for (int k = 0; k < n; k += B8 * SP) {   // (B8 SP divides kJoin)
#pragma unroll
      for (int i = 0; i < B8; ++i) {
        const int kk = k + SP * i + share;
        const float w = kk < n ? s_w[kk][row] : 0.f;
        // (weight 0: a piece without keys wrote no block, or one that is nothing beside the others)
        v.x += w == 0.f ? 0.f : a8[i].x * w;
        v.y += w == 0.f ? 0.f : a8[i].y * w;
        v.z += w == 0.f ? 0.f : a8[i].z * w;
        v.w += w == 0.f ? 0.f : a8[i].w * w;
      }
      if (k0 + k + B8 * SP < np) ask(k0 + k + B8 * SP);
    }
  }
  for (int off = NR; off < 32; off <<= 1) {
    v.x += __shfl_xor(v.x, off, 64);
    v.y += __shfl_xor(v.y, off, 64);
    v.z += __shfl_xor(v.z, off, 64);
    v.w += __shfl_xor(v.w, off, 64);
  }
  const float inv = row_factor(s_m[row], s_l[row]);
  store4(&s_out[row][4 * (tid >> 5)], v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  __syncthreads();
  if (tid >= 128) return;
  const int r = tid >> 2, d = tid % 4 * 8;   // 64 bytes a row
  if (r0 + r < rows)
    *reinterpret_cast<u32x4*>(out_row(p, tile.z, tile.w, r0 + r + head0) + 32 * t + d) = *reinterpret_cast<const u32x4*>(&s_out[r][d]);
}

// Which kernel runs, and its tiles: calls of at most 32 query rows per kv head
// and request (decode, verify) split each piece's keys over the waves and read
// them straight into registers; others share K and V tiles through LDS.
struct AttnPlan {
  bool few;
  int RT, P, G, min_share, step, tile_cost;
};
inline AttnPlan attn_plan(int Hq, int Hkv, int D, int max_rows) {
  const int rep = Hq / Hkv;
  AttnPlan a;
  a.few = max_rows > 0 && (long long)max_rows * rep <= 32;
  a.RT = a.few ? 32 : D == 256 ? 128 : 256;   // chunk_waves<D>() * 32
  a.P = (a.RT + rep - 2) / rep + 1;
  a.G = a.few ? device_cus() * (D < 256 ? 2 : 1) : device_cus() / 8 * 8;   // (chunks: dealt to eight XCDs)
  if (a.G < 8) a.G = 8;
  a.min_share = a.few ? 4 * kBlk : 2 * kStepKeys;
  a.step = a.few ? kBlk : kStepKeys;
  a.tile_cost = a.few ? 0 : 2 * kStepKeys;
  return a;
}

template <int D, int BITS>
int launch_attn(const PAttn& p, const AttnPlan& a, hipStream_t st) {
  constexpr int NW = chunk_waves<D>();
  if (a.few)
    hipLaunchKernelGGL((attn_few_kernel<D, BITS>), dim3((unsigned)p.G), dim3(kPT), 0, st, p);
  else
    hipLaunchKernelGGL((attn_chunk_kernel<D, BITS>), dim3((unsigned)p.G), dim3(64 * NW), 0, st, p);
  const int rc = launch_check("mtp_paged_attn");
  if (rc) return rc;
  const int blocks = a.RT / 32 * (D / 32);
  if (a.few)
    hipLaunchKernelGGL((attn_join_kernel<D, 32>), dim3((unsigned)p.G, blocks), dim3(kPT), 0, st, p);
  else
    hipLaunchKernelGGL((attn_join_kernel<D, 32 * NW>), dim3((unsigned)p.G, blocks), dim3(kPT), 0, st, p);
  return launch_check("mtp_paged_attn");
}

}  // namespace mtp

using namespace mtp;

MTP_API size_t mtp_paged_attn_workspace_bytes(int Hq, int Hkv, int D, int max_rows) {
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 1) return 0;
  const AttnPlan a = attn_plan(Hq, Hkv, D, max_rows);
  return (size_t)2 * a.G * a.RT * (D + 2) * sizeof(float) + (size_t)a.G * 16;
}

MTP_API int mtp_paged_attn(const mtp_paged_attn_args* a, void* stream) {
  const char* who = "mtp_paged_attn";
  if (!a || !a->q || !a->out || !a->k_pages || !a->v_pages || !a->block_table || !a->q_start || a->T < 1 ||
      a->Hkv < 1 || a->Hq < 1 || (a->bits == 8 && (!a->k_scales || !a->v_scales))) {
    set_error("%s: bad arguments", who);
    return MTP_ERR_ARG;
  }
  int rc = check_pages(who, a->D, a->page_size, a->num_pages, a->width, a->bits, a->B, a->Hkv);
  if (rc) return rc;
  if (a->Hq % a->Hkv || a->Hq / a->Hkv > 32) {
    set_error("%s: Hq=%d must be 1 to 32 times Hkv=%d", who, a->Hq, a->Hkv);
    return MTP_ERR_UNSUPPORTED;
  }
  if (!a->row_off && a->T % a->B) {
    set_error("%s: %d tokens are no whole rows of %d requests (give row_off)", who, a->T, a->B);
    return MTP_ERR_ARG;
  }
  if ((long long)a->T * a->Hq > 0x7fffffffLL) {
    set_error("%s: %d tokens of %d heads are more than 2^31 - 1 rows", who, a->T, a->Hq);
    return MTP_ERR_UNSUPPORTED;
  }
  if (!(a->scale > 0.f) || !(a->scale < 3.0e38f)) {
    set_error("%s: the scale must be positive and finite", who);
    return MTP_ERR_ARG;
  }
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->k_pages) || !aligned16(a->v_pages) ||
      !aligned16(a->k_scales) || !aligned16(a->v_scales) || !row_strides(a->q_token, a->q_head, a->D) ||
      !row_strides(a->out_token, a->out_head, a->D)) {
    set_error("%s: rows must be 16-byte aligned, their strides multiples of 8 elements", who);
    return MTP_ERR_ARG;
  }
  const int max_rows = a->row_off ? a->max_rows : a->T / a->B;
  const AttnPlan plan = attn_plan(a->Hq, a->Hkv, a->D, max_rows);
  const size_t need = mtp_paged_attn_workspace_bytes(a->Hq, a->Hkv, a->D, max_rows);
  if (!a->ws || !aligned16(a->ws) || a->ws_bytes < need) {
    set_error("%s: workspace %zu B < required %zu B (or unaligned)", who, a->ws_bytes, need);
    return MTP_ERR_WORKSPACE;
  }
  PAttn p = {};
  p.q = (const uint16_t*)a->q;
  p.out = (uint16_t*)a->out;
  p.k_pages = (const unsigned char*)a->k_pages;
  p.v_pages = (const unsigned char*)a->v_pages;
  p.k_scales = (const float*)a->k_scales;
  p.v_scales = (const float*)a->v_scales;
  p.table = a->block_table;
  p.q_start = a->q_start;
  p.row_off = a->row_off;
  p.status = a->status;
  p.part_o = (float*)a->ws;
  p.part_ml = p.part_o + (size_t)2 * plan.G * plan.RT * a->D;
  p.begun = reinterpret_cast<int4*>(p.part_ml + (size_t)2 * plan.G * plan.RT * 2);
  p.T = a->T;
  p.B = a->B;
  p.width = a->width;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.rep = a->Hq / a->Hkv;
  p.rep_inv = 65536u / (uint32_t)p.rep + 1;   // (exact while row * rep < 65536)
  p.bpp = a->page_size / kBlk;
  p.num_pages = a->num_pages;
  p.P = plan.P;
  p.rt_log2 = plan.RT == 32 ? 5 : plan.RT == 128 ? 7 : 8;
  p.G = plan.G;
  p.min_share = plan.min_share;
  p.step = plan.step;
  p.tile_cost = plan.tile_cost;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.out_token = a->out_token;
  p.out_head = a->out_head;
  hipStream_t st = (hipStream_t)stream;
  switch (a->D * 100 + a->bits) {
    case 6416: return launch_attn<64, 16>(p, plan, st);
    case 6408: return launch_attn<64, 8>(p, plan, st);
    case 12816: return launch_attn<128, 16>(p, plan, st);
    case 12808: return launch_attn<128, 8>(p, plan, st);
    case 25616: return launch_attn<256, 16>(p, plan, st);
    default: return launch_attn<256, 8>(p, plan, st);
  }
}
