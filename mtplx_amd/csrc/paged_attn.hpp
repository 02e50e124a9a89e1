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
// P is rounded to bf16 (as the values of V are; times their scale at 8 bits), l
// sums it before that: a weight is off by up to half a step, 2^-8 of it, each its
// own way, so a row over many keys by nearly as much as its output's own rounding
// (relative error against 64 bits 0.0022 where weights of 32 bits give 0.0017; 0.0026
// and 0.0020 at 8 bits). A P of two bf16 parts would keep it, for half as many matrix
// instructions again.
//
// Work is dealt by keys: every (request, kv head, row tile) is as long as the
// keys it sees plus a fixed cost, and workgroup g takes the g-th equal share
// of the whole line, whatever the lengths are. A tile that falls to more than
// one workgroup leaves one partial (o, m, l) per piece, at most two per
// workgroup, and attn_join adds them in the line's order. The split depends on
// lengths alone, so results do not depend on timing.
//
// Two more scopes share the kernels (each compiled in a source of its own):
//
// A window, with sinks: position p sees j > p - W and j < S. A tile's key blocks
// are those that hold sinks and those from its first row's window on, counted
// through without the gap between them; what is counted is dealt, loaded and
// masked as before, and what is not is never read. Every row's keys of a block are
// one range, so a mask is a word of bits per row and block.
//
// A shared prefix: paged_attn_shared.hip.
//
// Few rows (a request's up to 256 per kv head) of both are dealt in equal pieces
// without a line (dealt_piece).
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
//   head dim 64: the chunk 115 us, the verify rows 76; head dim 256: 1041 (16
//     bits: registers spill inside the step) and 529 (8 bits), the verify rows 230;
//   one token over 4k: 17.3 us, of which the two launches' kernels are 12 and 5;
//   behind a window of 4096 one token at 32k 14.8 us replayed (kernels 11.7 and
//     4.2, of which the keys' bytes are 3.2: a wave has one block of 32 keys, and
//     positions, queries, block table, keys, the waves' join, the partials and the
//     second launch's come one after another), sixteen requests' four verify rows 37
//     (8 bits, 140 MB in 31 us of the first kernel);
//   two requests of 256 rows behind a window of 2048: 48 and 10 us. 80 tiles over
//     256 CUs are twelve steps a workgroup, 23 us; the rest is their starts and 54 MB
//     of partials, which the join reads again (MFMAs 24% of the busy cycles);
//   a prompt of 8192 behind a window of 1024: 230 us, 700 TFLOP/s of what the
//     window leaves. A step of 64 keys is 2 us, as in the chunk, and a tile of 18
//     steps costs about 10 more: its rows' and first keys' way from memory, 1700
//     instructions of addresses, and three or four steps at the window's ends
//     whose masks are as many instructions as the softmax.
#pragma once

#include "paged.hpp"
#include "qmv_common.hpp"

#include <float.h>

#include <type_traits>

namespace mtp {

constexpr int kPT = 256;   // threads: four waves

// What a row sees of its request.
enum Scope {
  kCausal,   // every key up to its own position
  kWindow,   // of these the last `window` and the first `sinks`
  kPrefix,   // rows of all requests as one list: the shared prefix, all of it
  kTail,     // every key up to its own position, of which the prefix is done
};

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
  int window, sinks;   // kWindow
  long long most;      // kWindow: most line that a tile takes
  int splits;          // few rows, kWindow and kTail: most pieces of a tile
  int tiles;           // and tiles of a request's head that are dealt
  // kPrefix, kTail: positions that requests which begin behind them share, keys of
  // the prefix (the whole blocks of these), its row tiles of a kv head, their rows,
  // the pieces that each is cut into by keys; kTail: their partials, laid out as
  // part_o and part_ml, slot (head, piece, tile).
  int shared, prefix, prefix_tiles, prefix_rt_log2, prefix_pieces;
  const float* prefix_o;
  const float* prefix_ml;
  float scale_log2;
  long long q_token, q_head, out_token, out_head;
};

// Token and head (of those that share a kv head) of a row of a tile's list.
__device__ __forceinline__ int row_token(const PAttn& p, int r) { return (int)(((uint32_t)r * p.rep_inv) >> 16); }

// -- the line of work -------------------------------------------------------------


struct Req {
  int lo, n;          // packed rows
  int skip;           // kTail: blocks of the prefix (start, keys and lengths count behind them)
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
// The same where no tile takes more than `most`. Where the first ones, which
// see less, are few, all count as the others: tiles then end where equal shares
// of whole tiles do.
__device__ __forceinline__ bool tiles_alike(long long q0, int n, long long most) { return q0 + n >= 4 * most; }
__device__ __forceinline__ long long tiles_len(long long q0, int n, int P, long long t, long long most) {
  if (q0 + n <= most) return tiles_len(q0, n, P, t);
  if (tiles_alike(q0, n, most)) return t * most;
  const long long room = most - q0, under = room > 0 ? (long long)((uint32_t)room / (uint32_t)P) : 0;   // (room < n)
  return t <= under ? tiles_len(q0, n, P, t) : tiles_len(q0, n, P, under) + (t - under) * most;
}
template <int SC>
__device__ __forceinline__ long long scope_len(const PAttn& p, long long q0, int n, long long t) {
  if constexpr (SC == kWindow) return tiles_len(q0, n, p.P, t, p.most);
  else return tiles_len(q0, n, p.P, t);
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
template <int SC>
__device__ __forceinline__ long long head_len(const PAttn& p, long long start, int n) {
  return scope_len<SC>(p, clamp_start(p, start), n, tile_count(p, n));
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

// Tokens whose rows make the prefix's list.
__device__ __forceinline__ int prefix_tokens(const PAttn& p) {
  const int n = p.row_off ? p.row_off[p.B] : p.T;
  return n < 0 ? 0 : n < p.T ? n : p.T;
}

// The request whose pages the prefix is read from: the first that has rows and
// begins behind what is shared (a free slot of a batch has neither keys nor pages,
// and one that begins inside, if only in the block that is cut, may hold other
// keys); -1: none.
__device__ __forceinline__ int prefix_request(const PAttn& p, int lane) {
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const bool has = b < p.B && req_rows(p.row_off, b, p.B, p.T).n > 0 && p.q_start[b] >= p.shared;
    const unsigned long long m = __ballot(has);
    if (m) return b0 + __ffsll((long long)m) - 1;
  }
  return -1;
}

// The prefix is done for a request that begins behind what is shared; one that does
// not, or whose rows are not among the list's, sees its keys from the first on. (The
// join adds the prefix to the tiles that were dealt: a request that brings more
// rows than were announced does without, too.)
__device__ __forceinline__ bool behind_prefix(const PAttn& p, const ReqRows& rows, long long start) {
  return start >= p.shared && rows.lo + rows.n <= prefix_tokens(p) &&
         (long long)rows.n * p.rep <= (long long)p.tiles << p.rt_log2;
}

// A lane's request of the line (64 requests at a time), its rows and length.
struct LaneReq {
  ReqRows rows;
  long long start, len;   // len: one head
};
template <int SC>
__device__ __forceinline__ LaneReq lane_req(const PAttn& p, int b) {
  LaneReq r = {{0, 0}, 0, 0};
  if (b < p.B) {
    r.rows = req_rows(p.row_off, b, p.B, p.T);
    r.start = p.q_start[b];
    r.len = head_len<SC>(p, r.start, r.rows.n);
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
template <int SC>
struct Line {
  long long W, S;
  int G;
  __device__ __forceinline__ Line(const PAttn& p, int lane) {
    W = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) W += p.Hkv * lane_req<SC>(p, b0 + lane).len;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) W += __shfl_xor(W, off, 64);
    W = uniform64(W);
    // Equal shares, a whole number of steps each, no shorter than min_share.
    const long long s = W > 0 ? (W - 1) / p.G + 1 : 0;
    S = s > p.min_share ? (s + p.step - 1) & -(long long)p.step : p.min_share;
    if constexpr (SC == kWindow) {
      // Whole tiles, if at most a twentieth of the workgroups' time is lost that way: a
      // tile cut in two starts twice, and its partials are written and joined. Prompts,
      // cut and whole, by tiles a workgroup and what is lost: 40 heads over 8 of 128,
      // 8192 rows behind 512 (5, nothing) 179 and 162 us, behind 1024 247 and 228; 16000
      // behind 1024 (10, 2%) 484 and 475; 5000 (3, 9%) 190 and 197; 12000 behind 4096 (7,
      // 15%) 998 and 1057; 4000 (3, 39%) 153 and 185. 16 over 4 of 64, 4000 behind 256
      // (1, 2%) 37 and 23, 8192 behind 512 (2, nothing) 62 and 49, 4000 behind 1024 (1,
      // 16%) 57 and 62. 24 over 4 of 256, 8192 behind 512 (6, nothing) 568 and 533, 6000
      // behind 2000 (4, 7%) 1059 and 1102.
      const long long q = div_small(W, p.G * p.most) + 1, row = p.G * p.most;
      const long long whole = (q - 1) * row == W ? q - 1 : q;
      if (whole > 0 && 20 * whole * row <= 21 * W) S = whole * p.most;
    }
    G = W > 0 ? div_small(W - 1, S) + 1 : 0;
  }
  __device__ __forceinline__ long long lo(int g) const { return g * S; }
  __device__ __forceinline__ long long hi(int g) const { return g + 1 < G ? (g + 1) * S : W; }
  __device__ __forceinline__ int owner(long long x) const { return div_small(x, S); }
  // The request that holds line position x.
  __device__ __forceinline__ int find(const PAttn& p, int lane, long long x, Req& r) const {
    long long carry = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const LaneReq q = lane_req<SC>(p, b0 + lane);
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

// The prefix's list has no line: workgroup g takes piece k of tile t of head h,
// g = (h pieces + k) tiles + t (tiles that read the same keys are neighbours).
template <>
struct Line<kPrefix> {
  int G;
  __device__ __forceinline__ Line(const PAttn& p, int) { G = p.Hkv * p.prefix_pieces * p.prefix_tiles; }
  __device__ __forceinline__ long long lo(int) const { return 0; }
  __device__ __forceinline__ long long hi(int) const { return 1; }
};

// One row tile of one head: where it lies on the line and what it is. Tiles are
// whole whatever the heads of a kv head: a token's rows may lie in two of them.
struct Tile {
  long long begin, len;   // line
  int h, t;               // kv head, row tile
  int tok, off, rows;     // its first row: token of the request, head of that token; its rows
  long long pos;          // position of its first token
  int nk;                 // keys it sees: [0, nk)
  // kWindow: of these, the blocks of 32 that hold sinks and those from the first
  // row's window on, counted through without the gap between them.
  int nsink;              // blocks of sinks
  int gap;                // from the count of a block behind the sinks to its place
  int nkeys;              // keys of the blocks counted, up to nk
};
// All but begin and h, from t.
template <int SC>
__device__ __forceinline__ void set_tile(const PAttn& p, const Req& r, Tile& u) {
  const int first = u.t << p.rt_log2;   // (rows of a call: below 2^31)
  const int left = r.n * p.rep - first;
  u.rows = left >> p.rt_log2 ? 1 << p.rt_log2 : left;
  u.tok = (int)((uint32_t)first / (uint32_t)p.rep);
  u.off = first - u.tok * p.rep;
  const long long cost = (long long)(u.t + 1) * p.P;
  u.len = clamp_start(p, r.start) + (cost < r.n ? cost : r.n);
  if (SC == kWindow && (u.len > p.most || tiles_alike(clamp_start(p, r.start), r.n, p.most))) u.len = p.most;
  u.pos = r.start + u.tok;
  const long long cap = (long long)p.width * p.bpp * kBlk - (SC == kTail ? r.skip * kBlk : 0);
  if constexpr (SC == kTail) u.gap = r.skip;
  const long long e = u.pos + row_token(p, u.off + u.rows - 1) + 1;
  u.nk = (int)(e < 0 ? 0 : e > cap ? cap : e);
  if constexpr (SC == kWindow) {
    const int s = p.sinks < u.nk ? p.sinks : u.nk;
    const long long w = u.pos - p.window + 1;
    const int lo = w < s ? s : w < u.nk ? (int)w : u.nk;   // keys [s, lo) are seen by none of its rows
    u.nsink = (s + kBlk - 1) / kBlk;
    u.gap = (lo >> 5) - u.nsink;
    u.nkeys = lo < u.nk ? u.nk - 32 * u.gap : s;
  }
}
template <int SC>
__device__ __forceinline__ Tile tile_at(const PAttn& p, const Req& r, long long x) {
  Tile u;
  const long long y = x - r.base;
  u.h = div_small(y, r.head);
  const long long z = y - u.h * r.head;
  const long long q0 = clamp_start(p, r.start);
  int a = 0, b = tile_count(p, r.n) - 1;   // the last tile that begins at or before z
  while (a < b) {
    const int m = (a + b + 1) >> 1;
    if (scope_len<SC>(p, q0, r.n, m) <= z) a = m; else b = m - 1;
  }
  u.t = a;
  u.begin = r.base + u.h * r.head + scope_len<SC>(p, q0, r.n, a);
  set_tile<SC>(p, r, u);
  return u;
}

// Few rows, kWindow and kTail: no line. Lengths are alike (a window's) or short (a
// tail's), so every tile is cut into pieces of the same number of keys,
// workgroup (request, head, tile, piece) takes one, and what a workgroup has to
// know of the others is that number. The line's search, a wave's first 1500
// instructions, took as long as a decode step's keys: one token behind a window
// of 4096 20.5 us by the line and 15.1 dealt, sixteen requests' verify rows 44 and
// 36, sixteen tails of up to 600 keys 26 and 18 (kernel).
template <int SC>
__device__ __forceinline__ long long dealt_keys(const PAttn& p, int b) {
  const ReqRows rows = req_rows(p.row_off, b, p.B, p.T);
  long long start = p.q_start[b];
  const long long cap = (long long)p.width * p.bpp * kBlk;
  if constexpr (SC == kTail) {
    if (behind_prefix(p, rows, start)) start -= p.prefix;
  }
  long long n = start + rows.n;
  n = n > cap ? cap : n;
  if constexpr (SC == kWindow) {
    const long long most = (long long)p.window + p.sinks + rows.n + 2 * kBlk;
    n = n < most ? n + kBlk : most;   // (a block may count twice)
  }
  return rows.n < 1 || n < 0 ? 0 : n;
}
// Most keys of a piece: what spreads all keys over the CUs, no less than a block
// for each wave, and no more pieces than there are workgroups for. Every tile
// ends with a piece that is not whole, half of one on average, and pieces that
// are one too many for the CUs cost a second round.
template <int SC>
__device__ __forceinline__ int dealt_piece(const PAttn& p, int lane) {
  long long sum = 0, top = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const long long n = b0 + lane < p.B ? dealt_keys<SC>(p, b0 + lane) : 0;
    sum += n;
    top = n > top ? n : top;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, 64);
    const long long o = __shfl_xor(top, off, 64);
    top = o > top ? o : top;
  }
  sum = uniform64(sum) * (p.Hkv * p.tiles);
  top = uniform64(top);
  const int units = p.B * p.Hkv * p.tiles, groups = units < p.G ? p.G - units / 2 : p.G / 2;
  const long long share = div_small(sum, groups) + 1, least = div_small(top, p.splits) + 1;
  const long long c = share > least ? share : least;
  return c <= p.min_share ? p.min_share : (int)((c + kBlk - 1) & -(long long)kBlk);
}

// Workgroup g's piece of the prefix: tile u of the list rq, keys [ka, kb). Its
// rows are at the prefix's last position, so each sees all of it.
__device__ __forceinline__ void prefix_piece(const PAttn& p, int g, Req& rq, Tile& u, int& ka, int& kb, int step) {
  const int v = g / p.prefix_tiles, k = v % p.prefix_pieces;
  u.h = v / p.prefix_pieces;
  u.t = g - v * p.prefix_tiles;
  rq.lo = 0;
  rq.n = prefix_tokens(p);
  const int first = u.t << p.rt_log2, left = rq.n * p.rep - first;
  u.rows = left >> p.rt_log2 > 0 ? 1 << p.rt_log2 : left;
  u.tok = (int)((uint32_t)first / (uint32_t)p.rep);
  u.off = first - u.tok * p.rep;
  const long long cap = (long long)p.width * p.bpp * kBlk;
  u.nk = p.prefix < cap ? p.prefix : (int)cap;
  u.pos = u.nk - 1;
  const int steps = (u.nk + step - 1) / step;
  ka = (int)((long long)steps * k / p.prefix_pieces) * step;
  kb = (int)((long long)steps * (k + 1) / p.prefix_pieces) * step;
  if (kb > u.nk) kb = u.nk;
}

// The tile after u on the line, in the same request.
template <int SC>
__device__ __forceinline__ void next_tile(const PAttn& p, const Req& r, Tile& u) {
  u.begin += u.len;
  ++u.t;
  if (u.t == tile_count(p, r.n)) {
    u.t = 0;
    ++u.h;
  }
  set_tile<SC>(p, r, u);
}

// Keys [0, key_at(x)) of the tile (kWindow: of the counted ones) lie before
// offset x of its line: whole steps of `step` keys.
template <int SC>
__device__ __forceinline__ int key_at(const Tile& u, long long x, int step) {
  const int n = SC == kWindow ? u.nkeys : u.nk;
  if (x >= u.len) return n;
  const long long k = x / step * step;
  return k < n ? (int)k : n;
}
// The place of a tile's v-th counted block.
template <int SC>
__device__ __forceinline__ int block_place(const Tile& u, int v) {
  if constexpr (SC == kWindow) return v < u.nsink ? v : v + u.gap;
  else if constexpr (SC == kTail) return v + u.gap;
  else return v;
}

// Keys of one block that rows may see: a lane's row sees those in
// [low, bound], of which none at or past end exist. In the sinks' blocks that is
// every sink up to its position, behind them its window without the sinks (a
// block that holds the last sinks and keys of a window comes twice).
struct Sight {
  int base;   // first key
  int end;
  bool sink;
};

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
  int low;     // kWindow: first one behind the sinks
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

// The keys of a block, counted from its first, that a lane's row sees: [lo, hi]
// (lo > hi: none).
struct Range {
  int lo, hi;
};
template <int D>
__device__ __forceinline__ Range seen(const RowState<D>& s, const Sight& g) {
  const int last = (s.bound < g.end - 1 ? s.bound : g.end - 1) - g.base;
  return {g.sink || s.low < g.base ? 0 : s.low - g.base, last < 31 ? last : 31};
}
template <int D>
__device__ __forceinline__ bool any_seen(const RowState<D>& s, const Sight& g) {
  const Range k = seen(s, g);
  return k.lo <= k.hi;
}

// Scores to weights (the second product's operand), the running maximum and
// sum. ks(j, r), vs(j, r): scales of the lane's key of score register r (8
// bits), ks already times scale_log2. MASK: the row sees keys up to its bound,
// of block j none at or past end[j].
// WIN: by what `sight` says of each block instead.
template <int D, int BITS, int KB, bool MASK, bool WIN, class KS, class VS>
__device__ __forceinline__ void soften(RowState<D>& s, f32x16 (&st)[KB], u32x4 (&w)[KB][2], int kt,
                                       const int (&end)[KB], const Sight (&sight)[KB], int h2, float scale_log2, KS ks,
                                       VS vs) {
  // 16 bits without a mask: the maximum is taken before the scale (positive),
  // and scale and maximum go into one FMA.
  constexpr bool RAW = BITS == 16 && !MASK;
  const int bound = s.bound - kt;
  // WIN: the keys that the row sees, a bit each, from its half's first on.
  uint32_t vis[KB];
  if constexpr (WIN && MASK) {
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const Range k = seen(s, sight[j]);
      vis[j] = k.hi < k.lo ? 0u : ((2u << k.hi) - 1u & ~((1u << k.lo) - 1u)) >> (4 * h2);   // (2 << 31 is 0)
    }
  }
  auto shown = [&](int j, int r) { return (uint32_t)__builtin_amdgcn_sbfe((int)vis[j], 8 * (r >> 2) + (r & 3), 1); };
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
      if constexpr (WIN && MASK) {
        const uint32_t m = shown(j, r);
        x = __uint_as_float((__float_as_uint(x) & m) | (0xff800000u & ~m));
      } else {
        if (MASK && hidden(j, r)) x = -INFINITY;
      }
      st[j][r] = x;
      top = __builtin_elementwise_maximum(top, x);   // (no quieting of each x; a NaN makes its row NaN)
    }
  top = max_halves(top);
  if (RAW) top *= scale_log2;
  // A row that sees a key (of a block the first, then) has a finite maximum, so
  // it ends with l = 0 and m finite where all its scores are -infinity: NaN.
  bool sees = !MASK;
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    if constexpr (WIN && MASK) sees = sees || any_seen(s, sight[j]);
    else sees = sees || (kt + 32 * j <= s.bound && kt + 32 * j < end[j]);
  }
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
        if constexpr (WIN && MASK) {
          a = __uint_as_float(__float_as_uint(a * va) & shown(j, r));
          b = __uint_as_float(__float_as_uint(b * vb) & shown(j, r + 1));
        } else {
          a = MASK && hidden(j, r) ? 0.f : a * va;   // (a hidden key's scale may be NaN; of one that is seen it shows)
          b = MASK && hidden(j, r + 1) ? 0.f : b * vb;
        }
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
// WIN: by `sight`.
template <int D, int BITS, bool MASK, bool WIN, class VO>
__device__ __forceinline__ void add_values(RowState<D>& s, const u32x4 (&w)[2], int kt, int end, const Sight& sight,
                                           int h2, VO vop, bool odd_values = true) {
  u32x4 keep0 = {}, keep1 = {};
  uint32_t odd = 0;
  if (MASK && BITS == 16 && WIN && !odd_values) {   // (known to be finite, all of them)
    keep0 = keep1 = ~u32x4{};
  } else if (MASK && BITS == 16) {
    const int n = WIN ? sight.end - sight.base : end - kt;   // keys that exist
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
      bool mine = false;
      if constexpr (WIN) {
        const Range k = seen(s, sight);
        mine = key >= k.lo && key <= k.hi;
      }
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        const u32x4 v = ((vop(t, 0) & low) | (vop(t, 1) & ~low)) & only;
        const f32x16 add = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v),
                                                                   __builtin_bit_cast(bf16x8, wn), f32x16{}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) s.o[t][i] += (WIN ? mine : kt + key <= s.bound) ? add[i] : 0.f;
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
  template <int SC>
  __device__ __forceinline__ void fill(const PAttn& p, int b, const Tile& u, int blk, int end, int lane) {
    first = blk;
    at = blk + lane < end ? (int)page_block(p.table, p.width, b, block_place<SC>(u, blk + lane), p.bpp, p.num_pages,
                                            p.Hkv, u.h, 1) : -1;
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
template <int D, int SC>
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
  if constexpr (SC == kWindow) {
    const long long w = pos - p.window + 1;
    s.low = w > p.sinks ? w < 0x7fffffff ? (int)w : 0x7fffffff : p.sinks;
  }
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

// What the prefix left for a row of its list: the pieces' partials.
struct PrefixRow {
  const float4* o;    // of piece 0, its (32 rows, 32 d) blocks from here on
  const float2* ml;
  size_t o_step, ml_step;   // to the next piece
};
template <int D>
__device__ __forceinline__ PrefixRow prefix_row(const PAttn& p, int h, int row) {   // row: of the prefix's list
  const int RT = 1 << p.prefix_rt_log2, t = row >> p.prefix_rt_log2, rr = row & (RT - 1);
  const size_t slot = (size_t)h * p.prefix_pieces * p.prefix_tiles + t;
  return {reinterpret_cast<const float4*>(p.prefix_o) + (slot * (RT / 32) + (rr >> 5)) * (D / 32) * 256 + (rr & 31),
          reinterpret_cast<const float2*>(p.prefix_ml) + slot * RT + rr, (size_t)p.prefix_tiles * RT * D / 4,
          (size_t)p.prefix_tiles * RT};
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

constexpr int kWithPrefix = 1 << 30;

// What the join needs to know of the tile that workgroup g begins and others
// finish (at most one).
template <int SC>
__device__ __forceinline__ void note_begun(const PAttn& p, const Line<SC>& line, const Req& rq, const Tile& u, int g) {
  const int last = line.owner(u.begin + u.len - 1);
  const int pieces = (last < line.G ? last : line.G - 1) - g + 1;
  p.begun[g] = make_int4(u.rows | u.off << 16, pieces, rq.lo + u.tok, u.h);
}

// The v-th counted block of a windowed tile; `absent`: it has no page.
__device__ __forceinline__ Sight block_sight(const PAttn& p, const Tile& u, int v, bool absent) {
  const bool sink = v < u.nsink;
  const int base = 32 * block_place<kWindow>(u, v);
  return {base, absent ? base : sink && p.sinks < u.nk ? p.sinks : u.nk, sink};
}

// Of a windowed tile, for rows at positions [first, last] (first no further
// than its last key): counted blocks [low, full) hide no key from any of them,
// those behind `last` hide all.
template <int SC>
struct Sights {
  int low, full, last;
  __device__ __forceinline__ Sights(const PAttn& p, const Tile& u, long long first, long long end) {
    const long long w = end - p.window + 1;                   // from here on all see every key
    const int from = w > p.sinks ? w < u.nk ? (int)w : u.nk : p.sinks < u.nk ? p.sinks : u.nk;
    const int whole = first + 1 > 0 ? (int)((first + 1) >> 5) : 0;   // blocks [0, whole) hide no later key
    low = (from + 31) / 32 - u.gap;
    if (low < u.nsink) low = u.nsink;
    full = whole - u.gap;
    // Whole blocks of sinks before the window's, seen by all: the same run.
    if (low == u.nsink && p.sinks % 32 == 0 && p.sinks <= first + 1) low = 0;
    if (full < low) full = low;
    const long long e = end < u.nk - 1 ? end : u.nk - 1;
    last = e < 0 ? -1 : (int)(e >> 5) - (e >= p.sinks ? u.gap : 0);
  }
};

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
template <int D, int BITS, int SC>
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
  // kWindow, 16 bits: whether V of a step's blocks has an element that is no
  // number, as the waves that stage it see it (each wave that needs to know
  // looked at all of it: as many instructions as the softmax).
  constexpr bool FLAGS = SC == kWindow && BITS == 16;
  __shared__ int s_odd[FLAGS ? 8 : 1][2];   // (of step n % 8; that of n + 4 is cleared with n's)
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Line<SC> line(p, lane);
  if (SC != kPrefix && tid == 0 && (int)blockIdx.x >= line.G) p.begun[blockIdx.x] = make_int4(0, 0, 0, 0);
  // Neighbours on the line share a head's keys: they go to one XCD (workgroups
  // are dealt to the eight in turn), whose L2 then serves them.
  const int per = cdiv(line.G, 8);
  const int g = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if ((int)blockIdx.x >> 3 >= per || g >= line.G) return;
  if (SC != kPrefix && tid == 0) p.begun[g] = make_int4(0, 0, 0, 0);
  const long long lo = line.lo(g), hi = line.hi(g);
  const int turn = NW == 8 && wave >= 4 ? 1 : 0;
  const uint32_t klds = lds_addr(lds), vlds = klds + KR * 4 * BE;
  Req rq;
  int b;
  Tile u;
  int ka, kb;
  if constexpr (SC == kPrefix) {
    b = prefix_request(p, lane);
    prefix_piece(p, g, rq, u, ka, kb, kStepKeys);
    if (b < 0 || u.rows <= 0) return;   // (nobody reads it; fewer tokens than the launch was sized for)
  } else {
    b = line.find(p, lane, lo, rq);
    u = tile_at<SC>(p, rq, lo);
  }
  for (long long x = lo; x < hi;) {
    bool starts = true, ends = false;
    if constexpr (SC == kPrefix) {
      x = hi;
    } else {
      if (x >= rq.base + p.Hkv * rq.head) {
        b = line.find(p, lane, x, rq);
        u = tile_at<SC>(p, rq, x);
      } else if (x >= u.begin + u.len) {
        next_tile<SC>(p, rq, u);
      }
      const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
      ka = key_at<SC>(u, x - u.begin, kStepKeys);
      kb = key_at<SC>(u, end - u.begin, kStepKeys);
      starts = x == u.begin;
      ends = end == u.begin + u.len;
      x = end;
      if (starts && !ends && tid == 0) note_begun(p, line, rq, u, g);
    }
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
    blocks.fill<SC>(p, b, u, ka >> 5, (kb + 31) >> 5, lane);
    const int nstep = (kb - ka + kStepKeys - 1) / kStepKeys;
    // Steps [nlow, nfull) hide no key from any of the wave's rows and have all
    // their pages; [0, nlow) and [nfull, nlive) hide some; the rest hides all.
    int nlow = 0, nfull = 0, nlive = 0;
    if constexpr (SC == kWindow) {
      const Sights<SC> w(p, u, wmin, wmax);
      if (w.last >= ka >> 5) nlive = w.last >= (kb + 31) >> 5 ? nstep : ((w.last - (ka >> 5)) >> 1) + 1;
      if (w.low > ka >> 5) nlow = (w.low - (ka >> 5) + 1) >> 1;
      if (w.full > ka >> 5) nfull = (w.full - (ka >> 5)) >> 1;
    } else {
      if (wmax >= ka) nlive = wmax >= kb ? nstep : (int)((wmax - ka) / kStepKeys) + 1;
      if (nlive > 0 && wmin + 1 - ka >= kStepKeys) nfull = (int)((wmin + 1 - ka) / kStepKeys);
    }
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
        blocks.fill<SC>(p, b, u, blk0 + 2 * from, blk1, lane);
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
    auto flag_v = [&](int n) {   // step n's V, on its way to LDS
      if constexpr (FLAGS) {
        typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
        if (tid < 2) s_odd[(n + 4) & 7][tid] = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u16x8 top = {};
          bool any = false;
#pragma unroll
          for (int i = 0; i < LD; ++i) {
            const int c = i * NT + wave * 64;
            if (2 * CB % NT && c >= 2 * CB) break;
            if ((CB % NT ? c >= CB : i * NT >= CB) != (j == 1)) continue;
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8, vr[i] & 0x7fff7fffu));
            any = true;
          }
          if (!any) continue;
          const u32x4 m = __builtin_bit_cast(u32x4, top) + 0x00800080u;
          if (__any((m.x | m.y | m.z | m.w) & 0x80008000u) && lane == 0) s_odd[n & 7][j] = 1;
        }
      }
    };
    auto store_k = [&](int n) {   // of step n (slot k1 when n is the next step)
      put(klds + k1 * (4 * BE), kr);
      if (BITS == 8 && tid < kStepKeys) {
        ksc[n & 3][tid] = kscale * p.scale_log2;
        vsc[n & 3][tid] = vscale;
      }
    };
    auto store_v = [&](int n) {   // of step n + 1 (two slots: n)
      put(vlds + (VR == 3 ? v2 : v1) * (4 * BE), vr);
      flag_v(n + VR - 2);
    };
    if (nstep > 0) {   // step 0 in LDS (its V on the way, of two slots), step 1 on its way
      load(0, false);
      load(0, true);
    }
    unsigned char* const mine = lds + wave * (32 * row_bytes<D>());   // (of no step: between pieces)
    RowState<D> s;
    take_rows<D, SC>(s, ql, p, u, row0, lane, mine);
    f32x16 st[2];
    u32x4 w[2][2];
    // At D = 256 and 16 bits, eight operands at a time: two blocks' whole ones
    // (128 registers) beside 192 of accumulators and queries and 64 of tiles on
    // their way did not fit, and the step spilled.
    constexpr bool HALVES = D == 256 && BITS == 16;
    u32x4 op[2][HALVES ? 8 : D / 16];
    // Operands from a ring slot: one address, offsets in the instructions.
    auto operands = [&](uint32_t lds, int ring) {
      uint32_t a = lds + ring * (4 * BE) + lane * 16;
      asm("" : "+v"(a));
      return reinterpret_cast<const lds_u32x4*>(a);
    };
    constexpr int OPS = HALVES ? 8 : D / 16;
    auto ask = [&](u32x4 (&to)[OPS], const lds_u32x4* from, int j) {   // the j-th so many of a step's
#pragma unroll
      for (int i = 0; i < OPS; ++i) to[i] = from[(j * OPS + i) * 64];
      __builtin_amdgcn_sched_barrier(0);
    };
    auto keys = [&] {
      const lds_u32x4* k = operands(klds, k0);
      scores<D, 2>(s, st, [&](int j, int i) { return k[(j * (D / 16) + i) * 64]; });
    };
    auto ends2 = [&](int n, int j) { return blocks.absent(blk0 + 2 * n + j) ? 0 : u.nk; };
    auto sight = [&](int n, int j) {   // (kWindow)
      if constexpr (SC == kWindow) return block_sight(p, u, blk0 + 2 * n + j, blocks.absent(blk0 + 2 * n + j));
      else return Sight{};
    };
    auto values = [&](int n) {   // of step n, masked; slot v0 when n is the last step
      const lds_u32x4* v = operands(vlds, v0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        add_values<D, BITS, true, SC == kWindow>(s, w[j], ka + n * kStepKeys + 32 * j, ends2(n, j), sight(n, j), h2,
                                                 [&](int t, int jj) { return v[(j * (D / 16) + 2 * t + jj) * 64]; },
                                                 FLAGS ? __builtin_amdgcn_readfirstlane(s_odd[n & 7][j]) != 0 : true);
    };
    // Both products of step n, no key hidden: each eight operands are asked for
    // eight matrix instructions ahead (left alone, the compiler reads one, waits
    // for it and multiplies); op[0] is in hand.
    auto products = [&](int n) {
      const lds_u32x4* v = operands(vlds, v0);
      const lds_u32x4* k = operands(klds, k0);
      if constexpr (HALVES) {   // quarters c of the step: half c % 2 of block c / 2's operands
        auto add = [&](const u32x4 (&from)[OPS], int c) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f32x16& o = s.o[4 * (c & 1) + i / 2];
            o = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, from[i]),
                                                        __builtin_bit_cast(bf16x8, w[c >> 1][i & 1]), o, 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        auto score = [&](const u32x4 (&from)[OPS], int c) {
          if (!(c & 1)) st[c >> 1] = f32x16{};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            st[c >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, from[i]),
                                                                 s.q[8 * (c & 1) + i], st[c >> 1], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        };
        ask(op[0], v, 0);
        ask(op[1], v, 1);
        add(op[0], 0);
        ask(op[0], v, 2);
        add(op[1], 1);
        ask(op[1], v, 3);
        add(op[0], 2);
        ask(op[0], k, 0);
        store_k(n + 1);
        add(op[1], 3);
        ask(op[1], k, 1);
        store_v(n);
        score(op[0], 0);
        ask(op[0], k, 2);
        score(op[1], 1);
        ask(op[1], k, 3);
        load_next(n);
        score(op[0], 2);
        score(op[1], 3);
      }
      if constexpr (!HALVES) {
        auto add = [&](const u32x4 (&from)[OPS], int j) {
          add_values<D, BITS, false, false>(s, w[j], 0, 0, Sight{}, h2, [&](int t, int jj) { return from[2 * t + jj]; });
          __builtin_amdgcn_sched_barrier(0);
        };
        auto score = [&](const u32x4 (&from)[OPS], int j) {
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
        store_v(n);
        score(op[0], 0);
        load_next(n);
        score(op[1], 1);
      }
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
      const Sight sights[2] = {MASK ? sight(n, 0) : Sight{}, MASK ? sight(n, 1) : Sight{}};
      soften<D, BITS, 2, MASK, SC == kWindow>(
          s, st, w, ka + n * kStepKeys, end, sights, h2, p.scale_log2,
          [&](int j, int r) { return kss[32 * j + 8 * (r >> 2) + (r & 3)]; },
          [&](int j, int r) { return vss[32 * j + 8 * (r >> 2) + (r & 3)]; });
    };
    auto look_ahead = [&] {   // the next products' first operands: V of the step just softened
      if (VR == 3) ask(op[0], operands(vlds, v0), 0);
    };
    constexpr std::true_type yes;
    constexpr std::false_type no;
    if (FLAGS && tid < 16) s_odd[tid >> 1][tid & 1] = 0;
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
        flag_v(0);
        load(1, true);
      }
      lds_barrier();
      auto stage = [&](int n) {   // what goes with step n's products
        store_k(n + 1);
        store_v(n);
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
      // they are. (A window's first steps may hide keys too.)
      int n = 0;
      if constexpr (SC == kWindow) {
        if (nlow > 0 && nlive > 0) {
          keys();
          stage(0);
          between();
          weights(0, yes);
          after();
          for (n = 1; n < nlow && n < nlive; ++n) {
            values(n - 1);
            keys();
            stage(n);
            between();
            weights(n, yes);
            after();
          }
          if (n < nfull) {
            values(n - 1);
            keys();
            stage(n);
            between();
            weights(n, no);
            after();
            look_ahead();
            for (++n; n < nfull; ++n) {
              cover(n - 1, n + 2);
              products(n);
              between();
              weights(n, no);
              after();
              look_ahead();
            }
          }
        }
      }
      if (n > 0) {   // (a window's)
      } else if (nfull > 0) {
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
      const size_t slot = SC == kPrefix ? (size_t)g : 2 * (size_t)g + (starts ? 1 : 0);
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
template <int D, int BITS, int SC>
__global__ __launch_bounds__(kPT, D == 256 ? 1 : 2) void attn_few_kernel(PAttn p) {
  constexpr int RT = 32;
  constexpr int BE = kBlk * D;
  constexpr int LD = D / 16 * (BITS / 8) / 2;   // 16-byte loads of a lane per block
  constexpr int OS = D + 4;                     // padded row: lanes of one store hit distinct banks
  __shared__ __attribute__((aligned(16))) float s_o[4][32 * OS];
  __shared__ float s_m[4][32], s_l[4][32];
  const int tid = threadIdx.x, lane = tid & 63, c32 = lane & 31, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr bool DEALT = SC != kCausal;
  const Line<DEALT ? kPrefix : SC> line(p, lane);   // (dealt: none)
  const int g = blockIdx.x;
  Req rq;
  int b, piece = 0, share = 0, unit = 0, tile0 = 0;   // dealt: piece, most keys of one, (request, kv head, tile)
  Tile u;
  long long lo = 0, hi = 0;
  if constexpr (DEALT) {
    share = dealt_piece<SC>(p, lane);
    // First pieces first: the last ones may not be there, and neighbours go to
    // different XCDs (with a head's pieces as neighbours, some XCDs had none).
    const int units = p.B * p.Hkv * p.tiles;
    piece = g / units;
    unit = g - piece * units;
    const int head = unit / p.tiles;
    tile0 = unit - head * p.tiles;
    b = head / p.Hkv;
    u.h = head - b * p.Hkv;
    const ReqRows rows = req_rows(p.row_off, b, p.B, p.T);
    rq.lo = rows.lo;
    rq.n = rows.n;
    rq.start = p.q_start[b];
    rq.skip = SC == kTail && behind_prefix(p, rows, rq.start) ? p.prefix / kBlk : 0;
    rq.start -= rq.skip * kBlk;
    // Its tile; the first one's workgroups take those of rows that were not
    // announced too, whole.
    lo = tile0;
    hi = tile_count(p, rq.n);
    if (tile0 > 0 && hi > tile0) hi = tile0 + 1;
    if (piece == 0 && tid == 0) p.begun[unit] = make_int4(0, 0, 0, 0);
  } else {
    if (tid == 0) p.begun[g] = make_int4(0, 0, 0, 0);
    if (g >= line.G) return;
    lo = line.lo(g);
    hi = line.hi(g);
    b = line.find(p, lane, lo, rq);
    u = tile_at<SC>(p, rq, lo);
  }
  for (long long x = lo; x < hi;) {
    int ka, kb;
    bool starts = true, ends = true;
    if constexpr (DEALT) {
      u.t = (int)x++;
      if (u.t != tile0 && (u.t < p.tiles || u.t % p.splits != piece)) continue;
      set_tile<SC>(p, rq, u);
      const int n = SC == kWindow ? u.nkeys : u.nk;
      ka = 0;
      kb = n;
      if (u.t == tile0) {
        int np = n > share ? div_small(n - 1, share) + 1 : 1, size = n;
        if (np > 1) {   // equal ones
          size = (div_small(n - 1, np) + kBlk) & -kBlk;
          np = div_small(n - 1, size) + 1;
        }
        if (piece >= np) continue;
        ka = piece * size;
        if (piece + 1 < np) kb = ka + size;
        starts = ends = np == 1 && !rq.skip;   // (else the join has it)
        if (!ends && piece == 0 && tid == 0)
          p.begun[unit] = make_int4(u.rows | u.off << 16, np | (rq.skip ? kWithPrefix : 0), rq.lo + u.tok, u.h);
      }
    } else {
      if (x >= rq.base + p.Hkv * rq.head) {
        b = line.find(p, lane, x, rq);
        u = tile_at<SC>(p, rq, x);
      } else if (x >= u.begin + u.len) {
        next_tile<SC>(p, rq, u);
      }
      const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
      ka = key_at<SC>(u, x - u.begin, kBlk);
      kb = key_at<SC>(u, end - u.begin, kBlk);
      starts = x == u.begin;
      ends = end == u.begin + u.len;
      x = end;
      if (starts && !ends && tid == 0) note_begun(p, line, rq, u, g);
    }
    const int rows = u.rows;
    RowLoads<D> q;
    ask_rows<D>(q, p, rq, u, 0, lane);
    const long long wmin = u.pos < u.nk - 1 ? u.pos : u.nk - 1;   // blocks up to it hide no key
    const int nblk = (kb - ka + kBlk - 1) / kBlk;
    const int b0 = (ka >> 5) + nblk * wave / 4, b1 = (ka >> 5) + nblk * (wave + 1) / 4;   // the wave's blocks
    BlockList blocks;
    if (b0 < b1) blocks.fill<SC>(p, b, u, b0, b1, lane);
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
    take_rows<D, SC>(s, q, p, u, 0, lane, reinterpret_cast<unsigned char*>(s_o[wave]));
    float* const scales = s_o[wave];   // 8 bits: a block's scales, on their way to the lanes that need them
    auto block = [&](int blk, auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      const int kt = 32 * blk;
      Sight sight[1] = {};
      if constexpr (SC == kWindow && MASK) sight[0] = block_sight(p, u, blk, false);
      if constexpr (BITS == 8) scales[lane] = h2 ? sc : sc * p.scale_log2;
      auto scale = [&](int r) { return scales[8 * (r >> 2) + 4 * h2 + (r & 3)]; };
      f32x16 st[1];
      u32x4 w[1][2];
      const int end1[1] = {u.nk};
      scores<D, 1>(s, st, [&](int, int i) {
        if constexpr (BITS == 16) return kr[i];
        else return (i & 1) ? widen8(kr[i >> 1].z, kr[i >> 1].w) : widen8(kr[i >> 1].x, kr[i >> 1].y);
      });
      soften<D, BITS, 1, MASK, SC == kWindow>(
          s, st, w, kt, end1, sight, h2, p.scale_log2, [&](int, int r) { return scale(r); },
          [&](int, int r) { return scale(r + 16); });
      if (BITS == 8) __builtin_amdgcn_sched_barrier(0);   // (V's integers are not widened before their turn)
      add_values<D, BITS, MASK, SC == kWindow>(s, w[0], kt, u.nk, sight[0], h2, [&](int t, int jj) {
        if constexpr (BITS == 16) return vr[2 * t + jj];
        else return jj ? widen8(vr[t].z, vr[t].w) : widen8(vr[t].x, vr[t].y);
      });
    };
    auto next = [&](int blk) {   // the block after blk, in its place
      if (blk + 1 >= blocks.first + 64 && blk + 1 < b1) blocks.fill<SC>(p, b, u, blk + 1, b1, lane);
      load(blk + 1);
    };
    // Blocks [bl, bf) hide no key and have their pages.
    int bl = b0, bf = wmin + 1 >= 0 ? (int)((wmin + 1) >> 5) : 0;
    if constexpr (SC == kWindow) {
      const Sights<SC> w(p, u, wmin, u.pos + row_token(p, rows - 1 + u.off));
      bl = w.low;
      bf = w.full;
    }
    if (bf > b1) bf = b1;
    int blk = b0;
    while (blk < b1) {
      // As far as this list knows.
      int to = blocks.first + blocks.present();
      if (to > bf) to = bf;
      if (SC == kWindow && blk < bl) to = blk;
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
    const int slot = DEALT ? unit * p.splits + piece : 2 * g + (starts ? 1 : 0);
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

// PRE: a tile whose request has the prefix behind it sums the prefix's pieces of
// its rows too, after its own.
// DEALT: pieces of few rows that were dealt without a line.
template <int D, int RT, bool PRE, bool DEALT>
__global__ __launch_bounds__(kPT) void attn_join_kernel(PAttn p) {
  constexpr int kJoin = join_round<RT>();
  __shared__ float s_w[kJoin][32], s_m[32], s_l[32];
  __shared__ __attribute__((aligned(16))) uint16_t s_out[32][32 + 8];
  const int tid = threadIdx.x;
  const int g = blockIdx.x;
  const int4 tile = p.begun[g];   // rows (0: none) and first head, pieces, first token, kv head
  const int rows = tile.x & 0xffff, head0 = tile.x >> 16;
  const int own = PRE ? tile.y & (kWithPrefix - 1) : tile.y, np = PRE && tile.y & kWithPrefix ? own + p.prefix_pieces : own;
  const int rb = blockIdx.y / (D / 32), t = blockIdx.y % (D / 32);
  const int r0 = 32 * rb;
  if (r0 >= rows) return;
  // Piece k's slot: the one that begins the tile is g's second.
  auto slot = [&](int k) { return DEALT ? (size_t)g * p.splits + k : (size_t)(2 * (g + k) + (k == 0 ? 1 : 0)); };
  int NR = 32;   // (chunks' tiles: always, so that the loop below is a plain one)
  while (RT == 32 && NR > 4 && rows - r0 <= NR / 2) NR >>= 1;
  const int SP = 32 / NR, row = tid & (NR - 1), share = (tid & 31) / NR;
  // The prefix's rows: those past the tile's last are its last again (never used).
  auto list_row = [&](int r) { return tile.z * p.rep + head0 + (r0 + r < rows ? r0 + r : rows - 1); };
  PrefixRow pr = {}, pw = {};
  if constexpr (PRE) {
    pr = prefix_row<D>(p, tile.w, list_row(row));
    pw = prefix_row<D>(p, tile.w, list_row(tid >> 3));
  }
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int B8 = RT == 32 ? 8 : 4;   // pieces whose blocks are in flight together
  float4 a8[B8];
  auto ask = [&](int k) {   // (the last piece again past the last: never used)
#pragma unroll
    for (int i = 0; i < B8; ++i) {
      int kk = k + SP * i + share;
      kk = kk < np ? kk : np - 1;
      if (PRE && kk >= own)
        a8[i] = pr.o[(kk - own) * pr.o_step + t * 256 + (tid & ~31)];
      else
        a8[i] = part_block<D>(p, slot(kk), RT, rb, t)[(tid & ~31) + row];
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
        if (live && k < n) {
          if (PRE && k0 + k >= own)
            a[i] = pw.ml[(k0 + k - own) * pw.ml_step];
          else
            a[i] = *reinterpret_cast<const float2*>(p.part_ml + (slot(k0 + k) * RT + r0 + rr) * 2);
        }
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
  int tiles;   // dealt: of a request's head
};
// `dealt`: a call with a window or a shared prefix, whose few rows go without a
// line: up to eight tiles of 32 rows of a request's head.
inline AttnPlan attn_plan(int Hq, int Hkv, int D, int max_rows, bool dealt = false) {
  const int rep = Hq / Hkv;
  const long long rows = (long long)max_rows * rep;
  AttnPlan a;
  a.few = rows > 0 && rows <= (dealt ? 256 : 32);
  a.tiles = a.few ? (int)(rows + 31) / 32 : 0;
  a.RT = a.few ? 32 : D == 256 ? 128 : 256;   // chunk_waves<D>() * 32
  a.P = (a.RT + rep - 2) / rep + 1;
  a.G = a.few ? device_cus() * (D < 256 ? 2 : 1) : device_cus() / 8 * 8;   // (chunks: dealt to eight XCDs)
  if (a.G < 8) a.G = 8;
  a.min_share = a.few ? 4 * kBlk : 2 * kStepKeys;
  a.step = a.few ? kBlk : kStepKeys;
  a.tile_cost = a.few ? 0 : 2 * kStepKeys;
  return a;
}

template <int D, int BITS, int SC>
int launch_attn(const char* who, const PAttn& p, const AttnPlan& a, hipStream_t st) {
  constexpr int NW = chunk_waves<D>();
  constexpr bool DEALT = SC != kCausal;
  const unsigned tiles = a.few && DEALT ? (unsigned)(p.B * p.Hkv * p.tiles) : (unsigned)p.G;
  const int blocks = a.RT / 32 * (D / 32);
  if (a.few) {
    hipLaunchKernelGGL((attn_few_kernel<D, BITS, SC>), dim3(DEALT ? tiles * p.splits : tiles), dim3(kPT), 0, st, p);
    const int rc = launch_check(who);
    if (rc || (SC == kWindow && p.splits == 1)) return rc;   // (every tile whole)
    hipLaunchKernelGGL((attn_join_kernel<D, 32, SC == kTail, DEALT>), dim3(tiles, blocks), dim3(kPT), 0, st, p);
  } else if constexpr (SC != kTail) {   // (a tail's rows are few)
    hipLaunchKernelGGL((attn_chunk_kernel<D, BITS, SC>), dim3(tiles), dim3(64 * NW), 0, st, p);
    const int rc = launch_check(who);
    if (rc) return rc;
    hipLaunchKernelGGL((attn_join_kernel<D, 32 * NW, false, false>), dim3(tiles, blocks), dim3(kPT), 0, st, p);
  }
  return launch_check(who);
}

// One scope's kernels (each has a source of its own: they compile side by side).
template <int SC>
int launch_scope(const char* who, const PAttn& p, const AttnPlan& a, int D, int bits, hipStream_t st) {
  switch (D * 100 + bits) {
    case 6416: return launch_attn<64, 16, SC>(who, p, a, st);
    case 6408: return launch_attn<64, 8, SC>(who, p, a, st);
    case 12816: return launch_attn<128, 16, SC>(who, p, a, st);
    case 12808: return launch_attn<128, 8, SC>(who, p, a, st);
    case 25616: return launch_attn<256, 16, SC>(who, p, a, st);
    default: return launch_attn<256, 8, SC>(who, p, a, st);
  }
}
int launch_window(const char* who, const PAttn& p, const AttnPlan& a, int D, int bits, hipStream_t st);

// Pieces that a tile may fall into when few rows are dealt: two rounds of
// workgroups at most (a piece that is not there costs its start).
inline int dealt_splits(const AttnPlan& a, int B, int Hkv) {
  const long long n = 2LL * a.G / ((long long)B * Hkv * a.tiles);
  return n < 1 ? 1 : n > 128 ? 128 : (int)n;
}
inline size_t dealt_slots(const AttnPlan& a, int B, int Hkv, bool shared) {
  const int n = dealt_splits(a, B, Hkv);
  return n == 1 && !shared ? 0 : (size_t)B * Hkv * a.tiles * n;   // (whole tiles leave no partials)
}
inline size_t scoped_bytes(const AttnPlan& a, int D, int B, int Hkv, bool shared) {
  const size_t slots = a.few ? dealt_slots(a, B, Hkv, shared) : 2 * (size_t)a.G;
  return slots * a.RT * (D + 2) * sizeof(float) + (a.few ? (size_t)B * Hkv * a.tiles : (size_t)a.G) * sizeof(int4);
}

// The shared prefix's row tiles of a kv head, and the pieces of keys that each
// falls into: about what fills the CUs, whole rounds of them.
struct PrefixPlan {
  int RT, tiles, pieces;
  size_t slots(int Hkv) const { return (size_t)Hkv * tiles * pieces; }
  size_t bytes(int Hkv, int D) const { return slots(Hkv) * RT * (D + 2) * sizeof(float); }
};
inline PrefixPlan prefix_plan(int Hq, int Hkv, int D, int T, int prefix) {
  PrefixPlan a;
  a.RT = D == 256 ? 128 : 256;
  a.tiles = (int)(((long long)T * (Hq / Hkv) + a.RT - 1) / a.RT);
  a.pieces = 1;
  const int cus = device_cus() / 8 * 8 > 0 ? device_cus() / 8 * 8 : 8, steps = (prefix + kStepKeys - 1) / kStepKeys;
  const long long units = (long long)Hkv * a.tiles;
  double best = 1e30;
  for (int np = 1; np <= 64 && np <= (steps + 1) / 2; ++np) {
    // Rounds of workgroups, each its steps and the cost of a start and an end (four
    // steps'); a piece's partial is read once more (an eighth of a step).
    const double cost = (double)((units * np + cus - 1) / cus) * ((steps + np - 1) / np + 4) + 0.125 * np;
    if (cost < best) {
      best = cost;
      a.pieces = np;
    }
  }
  return a;
}
int launch_shared(const char* who, PAttn p, const AttnPlan& a, const PrefixPlan& pre, int D, int bits, hipStream_t st);

}  // namespace mtp
