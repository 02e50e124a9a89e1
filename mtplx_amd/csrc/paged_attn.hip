// Causal attention of new tokens over the paged KV cache, from one decoded row
// per request to whole prompts, mixed as they come.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= position of i,
//
// in one pass over the keys with the running maximum m and sum l of each row:
// a block of scores s gives p = 2^(s log2e scale - m), l += sum p, o += p v.
// m moves only when a block's maximum passes it by 8 (then o and l are scaled
// by 2^(old - new)): p stays below 2^8 and fp32 carries the rest, and most
// blocks cost no pass over o.
//
// The query rows of the heads that share a kv head are one list per request
// (row r = token r / rep, head r % rep), so K and V are read once for all of
// them. S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16_bf16: a lane
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
#include "paged.hpp"

namespace mtp {

constexpr int kPT = 256;   // threads: four waves

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
  int T, B, width, Hq, Hkv, rep, bpp, num_pages;
  int P;            // tokens of a row tile
  int G;            // most workgroups
  int min_share;    // least keys of a workgroup's share
  float scale_log2;
  long long q_token, q_head, out_token, out_head;
};

// -- the line of work -------------------------------------------------------------

constexpr int kTileCost = 64;   // keys' worth of a row tile's own cost (Q in, O out)

struct Req {
  int lo, n;          // packed rows
  long long start;    // position of the first
  long long base;     // line position where its first head begins
  long long head;     // line length of one head
};

// Line length of a request's first t row tiles (one head).
__device__ __forceinline__ long long tiles_len(long long q0, int n, int P, long long t) {
  // sum over tiles x < t of q0 + min((x + 1) P, n) + kTileCost
  const long long full = n / P;
  const long long f = t < full ? t : full;
  return t * (q0 + kTileCost) + P * (f * (f + 1) / 2) + (t - f) * n;
}
__device__ __forceinline__ long long clamp_start(const PAttn& p, long long s) {
  const long long cap = (long long)p.width * p.bpp * kBlk;
  return s < 0 ? 0 : s > cap ? cap : s;
}
__device__ __forceinline__ long long head_len(const PAttn& p, long long start, int n) {
  return tiles_len(clamp_start(p, start), n, p.P, (n + p.P - 1) / p.P);
}

__device__ __forceinline__ long long shfl64(long long v, int src) { return __shfl(v, src, 64); }

// Total length of the line, and the request that holds line position x (by
// scans of 64 requests at a time; every wave for itself).
__device__ __forceinline__ long long line_total(const PAttn& p, int lane) {
  long long sum = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    long long v = 0;
    const int b = b0 + lane;
    if (b < p.B) v = p.Hkv * head_len(p, p.q_start[b], req_rows(p.row_off, b, p.B, p.T).n);
    sum += v;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  return sum;
}

__device__ __forceinline__ int find_req(const PAttn& p, int lane, long long x, Req& r) {
  long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    long long len = 0, start = 0;
    ReqRows rr = {0, 0};
    if (b < p.B) {
      rr = req_rows(p.row_off, b, p.B, p.T);
      start = p.q_start[b];
      len = head_len(p, start, rr.n);
    }
    long long incl = p.Hkv * len;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const long long t = __shfl_up(incl, off, 64);
      if (lane >= off) incl += t;
    }
    const unsigned long long m = __ballot(len > 0 && x < carry + incl);   // the first whose end lies behind x
    if (m) {
      const int src = __ffsll((long long)m) - 1;
      r.lo = __builtin_amdgcn_readfirstlane(__shfl(rr.lo, src, 64));
      r.n = __builtin_amdgcn_readfirstlane(__shfl(rr.n, src, 64));
      r.start = shfl64(start, src);
      r.head = shfl64(len, src);
      r.base = carry + shfl64(incl, src) - p.Hkv * r.head;
      return __builtin_amdgcn_readfirstlane(b0 + src);
    }
    carry += shfl64(incl, 63);
  }
  return -1;
}

// Shares of the line: workgroup g of G takes [lo(g), lo(g + 1)).
struct Shares {
  long long W;
  int G;
  __device__ Shares(long long W_, int most, int min_share) : W(W_) {
    const long long n = W_ / min_share;
    G = n < 1 ? 1 : n < most ? (int)n : most;
  }
  __device__ long long lo(int g) const { return (long long)g * W / G; }
  __device__ int owner(long long x) const { return (int)(((x + 1) * G - 1) / W); }
};

// One row tile of one head: where it lies on the line and what it is.
struct Tile {
  long long begin, len;   // line
  int h, t;               // kv head, row tile
  int n;                  // its tokens
  long long pos;          // position of its first token
  int nk;                 // keys it sees: [0, nk)
};
__device__ __forceinline__ Tile tile_at(const PAttn& p, const Req& r, long long x) {
  Tile u;
  const long long y = x - r.base;
  u.h = (int)(y / r.head);
  const long long z = y - u.h * r.head;
  const long long q0 = clamp_start(p, r.start);
  int a = 0, b = (r.n + p.P - 1) / p.P - 1;   // the last tile that begins at or before z
  while (a < b) {
    const int m = (a + b + 1) >> 1;
    if (tiles_len(q0, r.n, p.P, m) <= z) a = m; else b = m - 1;
  }
  u.t = a;
  const long long z0 = tiles_len(q0, r.n, p.P, a);
  u.begin = r.base + u.h * r.head + z0;
  u.len = tiles_len(q0, r.n, p.P, a + 1) - z0;
  u.n = r.n - a * p.P < p.P ? r.n - a * p.P : p.P;
  u.pos = r.start + (long long)a * p.P;
  const long long cap = (long long)p.width * p.bpp * kBlk;
  const long long e = u.pos + u.n;
  u.nk = (int)(e < 0 ? 0 : e > cap ? cap : e);
  return u;
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

template <int D, int NB>
struct RowState {
  bf16x8 q[NB][D / 16];
  f32x16 o[NB][D / 32];
  float m[NB], l[NB];
  int bound[NB];   // last key that the lane's row sees; -1: no row here
};

// Keys (bit k: key kt + k) of a 16-bit V block with a NaN or an infinity in
// any element; the same in every lane.
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

// kop(i), vop(t, jj): operands (bf16, the latter as their 16 bytes); ks(r), vs(r): scales of the lane's key of
// score register r (8 bits), ks already times scale_log2. Keys kt..kt+31.
template <int D, int BITS, int NB, bool MASK, class KO, class VO, class KS, class VS>
__device__ __forceinline__ void attend(RowState<D, NB>& s, int kt, int h2, float scale_log2, KO kop, VO vop, KS ks,
                                       VS vs) {
  f32x16 st[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) st[n] = f32x16{};
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const bf16x8 k = kop(i);
#pragma unroll
    for (int n = 0; n < NB; ++n) st[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, s.q[n][i], st[n], 0, 0, 0);
  }
  bf16x8 w[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float x[16];
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = BITS == 8 ? st[n][r] * ks(r) : st[n][r] * scale_log2;
      if (MASK) {
        const int key = kt + 8 * (r >> 2) + 4 * h2 + (r & 3);
        x[r] = key <= s.bound[n] ? x[r] : -INFINITY;
      }
      top = fmaxf(top, x[r]);
    }
    top = max_halves(top);
    if (__any(top > s.m[n] + 8.f)) {
      // Only the rows that passed: the others' bits do not turn on their neighbours.
      const float m_new = top > s.m[n] + 8.f ? top : s.m[n];
      const float corr = s.m[n] == -INFINITY ? 0.f : exp2_fast(s.m[n] - m_new);
      s.m[n] = m_new;
      s.l[n] *= corr;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s.o[n][t][r] *= corr;
    }
    const float m = s.m[n] == -INFINITY ? 0.f : s.m[n];
    float sum = 0.f;
    uint32_t pk[8];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      float a = exp2_fast(x[r] - m), b = exp2_fast(x[r + 1] - m);
      sum += a + b;
      if (BITS == 8) {
        const float va = vs(r), vb = vs(r + 1);
        a = MASK && a == 0.f ? 0.f : a * va;   // a hidden key's scale may be NaN
        b = MASK && b == 0.f ? 0.f : b * vb;
      }
      pk[r / 2] = f2bf2(a, b);
    }
    s.l[n] += sum;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
      w[n][jj] = __builtin_bit_cast(bf16x8, u32x4{pk[4 * jj], pk[4 * jj + 1], pk[4 * jj + 2], pk[4 * jj + 3]});
  }
  // A hidden key's weight is 0, but 0 times a NaN or an infinity in its value is
  // not: in blocks with hidden keys (MASK), keys whose values are not all
  // finite leave the product and are added one by one, to the rows that see them.
  // (8-bit values are integers; their scale went into the weight.)
  u32x4 keep0 = {}, keep1 = {};
  uint32_t odd = 0;
  if (MASK && BITS == 16) {
    odd = odd_keys<D>(vop, h2);
    auto word = [&](int jj, int i) {
      return (odd >> (16 * jj + v_slot_key(h2, 2 * i)) & 1 ? 0u : 0x0000ffffu) |
             (odd >> (16 * jj + v_slot_key(h2, 2 * i + 1)) & 1 ? 0u : 0xffff0000u);
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
#pragma unroll
      for (int n = 0; n < NB; ++n)
        s.o[n][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), w[n][jj], s.o[n][t], 0, 0, 0);
    }
  if (MASK && BITS == 16) {
    for (; odd; odd &= odd - 1) {
      const int key = __ffs((int)odd) - 1, r = key & 15;
      const int e = r < 8 ? (r & 3) : 4 + (r & 3);
      const uint32_t half = h2 != (r & 7) >> 2 ? 0u : e & 1 ? 0xffff0000u : 0x0000ffffu;
      const int word = e >> 1;
      const u32x4 only = {word == 0 ? half : 0u, word == 1 ? half : 0u, word == 2 ? half : 0u, word == 3 ? half : 0u};
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        const u32x4 v = (key < 16 ? vop(t, 0) : vop(t, 1)) & only;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const bf16x8 wn = key < 16 ? w[n][0] : w[n][1];
          const f32x16 add = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), wn, f32x16{}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) s.o[n][t][i] += kt + key <= s.bound[n] ? add[i] : 0.f;
        }
      }
    }
  }
}

// Rows of the wave's NB blocks of 32: query operands, bounds; every row of the
// list is (token r / rep, head r % rep).
template <int D, int NB>
__device__ __forceinline__ void load_rows(RowState<D, NB>& s, const PAttn& p, const Req& rq, const Tile& u, int row0,
                                          int lane) {
  const int c = lane & 31, h2 = lane >> 5;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int r = row0 + 32 * n + c;
    const int i = r / p.rep, g = r - i * p.rep;
    const bool valid = i < u.n;
    const long long pos = u.pos + i;
    s.bound[n] = !valid || pos < 0 ? -1 : pos < u.nk ? (int)pos : u.nk - 1;
    const long long tok = rq.lo + (long long)u.t * p.P + (valid ? i : 0);
    const uint16_t* row = p.q + tok * p.q_token + (long long)(u.h * p.rep + (valid ? g : 0)) * p.q_head;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const u32x4 raw = *reinterpret_cast<const u32x4*>(row + (D / 2) * h2 + 8 * j);
      s.q[n][j] = __builtin_bit_cast(bf16x8, valid ? raw : u32x4{0, 0, 0, 0});
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t) s.o[n][t] = f32x16{};
    s.m[n] = -INFINITY;
    s.l[n] = 0.f;
  }
}

// 16 bytes read once per launch (non-temporal, as ld_stream).
__device__ __forceinline__ u32x4 ld_nt(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// Four consecutive d of an output row.
__device__ __forceinline__ void store4(uint16_t* dst, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(f2bf2(a, b), f2bf2(c, d));
}

__device__ __forceinline__ uint16_t* out_row(const PAttn& p, const Req& rq, const Tile& u, int r) {
  const int i = r / p.rep, g = r - i * p.rep;
  return p.out + (rq.lo + (long long)u.t * p.P + i) * p.out_token + (long long)(u.h * p.rep + g) * p.out_head;
}

// Eight bytes of integers -> eight bf16 (exact).
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  auto pair = [](uint32_t w, int i) {
    return f2bf2((float)(int8_t)(w >> (8 * i)), (float)(int8_t)(w >> (8 * i + 8)));
  };
  return u32x4{pair(a, 0), pair(a, 2), pair(b, 0), pair(b, 2)};
}

// V operand registers (keys 16 jj + v_slot_key(h2, .) of block key kt) with the keys at
// or past nk zeroed: stale bits of a page's tail are no numbers.
__device__ __forceinline__ u32x4 cut_tail(u32x4 v, int key0, int h2, int nk) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = key0 + v_slot_key(h2, 2 * i) < nk ? 0x0000ffffu : 0u;
    const uint32_t hi = key0 + v_slot_key(h2, 2 * i + 1) < nk ? 0xffff0000u : 0u;
    v[i] &= lo | hi;
  }
  return v;
}

// -- chunks: row tiles of 128 NB rows, K and V tiles shared through LDS ----------

constexpr int kStepKeys = 64;

template <int D, int BITS, int NB>
__global__ __launch_bounds__(kPT, 1) void attn_chunk_kernel(PAttn p) {
  constexpr int RT = 4 * 32 * NB;
  constexpr int BE = kBlk * D;                    // elements of a block
  constexpr int CB = BE * (BITS / 8) / 16;        // 16-byte chunks of a block
  constexpr int LD = 2 * CB / kPT;                // a thread's, of a step's two blocks
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][2 * BE];
  __shared__ __attribute__((aligned(16))) uint16_t vbuf[2][2 * BE];
  __shared__ __attribute__((aligned(16))) float ksc[2][kStepKeys], vsc[2][kStepKeys];
  const int tid = threadIdx.x, lane = tid & 63, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shares sh(line_total(p, lane), p.G, p.min_share);
  const int g = blockIdx.x;
  if (sh.W == 0 || g >= sh.G) return;
  const long long lo = sh.lo(g), hi = sh.lo(g + 1);
  Req rq;
  int b = find_req(p, lane, lo, rq);
  for (long long x = lo; x < hi;) {
    if (x >= rq.base + p.Hkv * rq.head) b = find_req(p, lane, x, rq);
    const Tile u = tile_at(p, rq, x);
    const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
    const int ka = key_at(u, x - u.begin, kStepKeys), kb = key_at(u, end - u.begin, kStepKeys);
    const bool starts = x == u.begin, ends = end == u.begin + u.len;
    x = end;
    const int row0 = wave * 32 * NB;
    const int rows = u.n * p.rep;   // of the tile
    RowState<D, NB> s;
    load_rows<D, NB>(s, p, rq, u, row0, lane);
    // Bounds of the wave's rows: blocks behind wmax are skipped, blocks up to
    // wmin need no mask (rows past the list are computed on zeros, and dropped).
    const int last = (row0 + 32 * NB < rows ? row0 + 32 * NB : rows) - 1;
    long long wmin = u.pos + row0 / p.rep, wmax = row0 < rows ? u.pos + last / p.rep : -1;
    if (wmin > u.nk - 1) wmin = u.nk - 1;

    u32x4 kr[LD], vr[LD];
    float kscale = 0.f, vscale = 0.f;
    long long at[2], nat[2];
    auto lookup = [&](int kt, long long (&a)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        a[j] = kt + 32 * j < kb ? page_block(p.table, p.width, b, (kt >> 5) + j, p.bpp, p.num_pages, p.Hkv, u.h, BE)
                                : -2;
    };
    auto load = [&](const long long (&a)[2]) {
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int c = i * kPT + tid;
        const long long at_j = c / CB ? a[1] : a[0];
        const size_t o = (size_t)(at_j < 0 ? 0 : at_j) * (BITS / 8) + (size_t)(c % CB) * 16;
        kr[i] = *reinterpret_cast<const u32x4*>(p.k_pages + o);
        vr[i] = *reinterpret_cast<const u32x4*>(p.v_pages + o);
      }
      if constexpr (BITS == 8) {
        if (tid < kStepKeys) {
          const long long a0 = tid < 32 ? a[0] : a[1];
          const size_t o = (size_t)(a0 < 0 ? 0 : a0) / D + (tid & 31);
          kscale = p.k_scales[o] * p.scale_log2;
          vscale = p.v_scales[o];
        }
      }
    };
    auto store = [&](int buf, int kt) {
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int c = i * kPT + tid, j = c / CB, cb = c % CB;
        if constexpr (BITS == 16) {
          *reinterpret_cast<u32x4*>(&kbuf[buf][c * 8]) = kr[i];
          u32x4 v = vr[i];
          if (kt + kStepKeys > u.nk) v = cut_tail(v, kt + 32 * j + 16 * ((cb >> 6) & 1), (cb >> 5) & 1, u.nk);
          *reinterpret_cast<u32x4*>(&vbuf[buf][c * 8]) = v;
        } else {
          const int o = j * BE + (2 * (cb >> 6) * 64 + (cb & 63)) * 8;
          *reinterpret_cast<u32x4*>(&kbuf[buf][o]) = widen8(kr[i].x, kr[i].y);
          *reinterpret_cast<u32x4*>(&kbuf[buf][o + 512]) = widen8(kr[i].z, kr[i].w);
          *reinterpret_cast<u32x4*>(&vbuf[buf][o]) = widen8(vr[i].x, vr[i].y);
          *reinterpret_cast<u32x4*>(&vbuf[buf][o + 512]) = widen8(vr[i].z, vr[i].w);
        }
      }
      if constexpr (BITS == 8) {
        if (tid < kStepKeys) {
          ksc[buf][tid] = kscale;
          vsc[buf][tid] = vscale;
        }
      }
    };
    if (ka < kb) {
      lookup(ka, at);
      load(at);
      lookup(ka + kStepKeys, nat);
      store(0, ka);
      __syncthreads();
      int buf = 0;
      for (int kt = ka; kt < kb; kt += kStepKeys) {
        const bool more = kt + kStepKeys < kb;
        const long long cur0 = at[0], cur1 = at[1];
        if (more) {
          at[0] = nat[0];
          at[1] = nat[1];
          load(at);
          lookup(kt + 2 * kStepKeys, nat);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k0 = kt + 32 * j;
          const long long here = j ? cur1 : cur0;
          if (here == -1 && p.status && tid == 0 && k0 < kb) atomicOr(p.status, kStatusPage);
          if (here < 0 || k0 > wmax) continue;   // uniform over the wave
          const uint16_t* kl = &kbuf[buf][j * BE + lane * 8];
          const uint16_t* vl = &vbuf[buf][j * BE + lane * 8];
          const float* kss = &ksc[buf][32 * j + 4 * h2];
          const float* vss = &vsc[buf][32 * j + 4 * h2];
          auto kop = [&](int i) { return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(kl + i * 512)); };
          auto vop = [&](int t, int jj) {
            return *reinterpret_cast<const u32x4*>(vl + (2 * t + jj) * 512);
          };
          auto ks = [&](int r) { return kss[8 * (r >> 2) + (r & 3)]; };
          auto vs = [&](int r) { return vss[8 * (r >> 2) + (r & 3)]; };
          if (k0 + 31 <= wmin)
            attend<D, BITS, NB, false>(s, k0, h2, p.scale_log2, kop, vop, ks, vs);
          else
            attend<D, BITS, NB, true>(s, k0, h2, p.scale_log2, kop, vop, ks, vs);
        }
        if (more) store(buf ^ 1, kt + kStepKeys);
        __syncthreads();
        buf ^= 1;
      }
    }
    // Out: the whole tile's rows, or this piece's partial.
    const int slot = 2 * g + (starts ? 1 : 0);
    const bool whole = starts && ends;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int r = row0 + 32 * n + (lane & 31);
      if (r >= rows) continue;
      const float l = s.l[n] + __shfl_xor(s.l[n], 32, 64);
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* dst = out_row(p, rq, u, r);
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            store4(dst + 32 * t + 8 * j + 4 * h2, s.o[n][t][4 * j] * inv, s.o[n][t][4 * j + 1] * inv,
                   s.o[n][t][4 * j + 2] * inv, s.o[n][t][4 * j + 3] * inv);
      } else if (ka < kb) {
        float* po = p.part_o + ((size_t)slot * RT + r) * D;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(po + 32 * t + 8 * j + 4 * h2) =
                make_float4(s.o[n][t][4 * j], s.o[n][t][4 * j + 1], s.o[n][t][4 * j + 2], s.o[n][t][4 * j + 3]);
        if (h2 == 0) {
          float* ml = p.part_ml + ((size_t)slot * RT + r) * 2;
          ml[0] = s.m[n];
          ml[1] = l;
        }
      }
    }
  }
}

// -- few rows: one tile of 32 rows, the four waves share a piece by keys ---------

template <int D, int BITS>
__global__ __launch_bounds__(kPT) void attn_few_kernel(PAttn p) {
  constexpr int RT = 32;
  constexpr int BE = kBlk * D;
  constexpr int LD = D / 16 * (BITS / 8) / 2;   // 16-byte loads of a lane per block
  constexpr int OS = D + 4;                     // padded row: lanes of one store hit distinct banks
  __shared__ __attribute__((aligned(16))) float s_o[4][32 * OS];
  __shared__ float s_m[4][32], s_l[4][32];
  const int tid = threadIdx.x, lane = tid & 63, c32 = lane & 31, h2 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shares sh(line_total(p, lane), p.G, p.min_share);
  const int g = blockIdx.x;
  if (sh.W == 0 || g >= sh.G) return;
  const long long lo = sh.lo(g), hi = sh.lo(g + 1);
  Req rq;
  int b = find_req(p, lane, lo, rq);
  for (long long x = lo; x < hi;) {
    if (x >= rq.base + p.Hkv * rq.head) b = find_req(p, lane, x, rq);
    const Tile u = tile_at(p, rq, x);
    const long long end = hi < u.begin + u.len ? hi : u.begin + u.len;
    const int ka = key_at(u, x - u.begin, kBlk), kb = key_at(u, end - u.begin, kBlk);
    const bool starts = x == u.begin, ends = end == u.begin + u.len;
    x = end;
    const int rows = u.n * p.rep;
    RowState<D, 1> s;
    load_rows<D, 1>(s, p, rq, u, 0, lane);
    const long long wmin = u.pos < u.nk - 1 ? u.pos : u.nk - 1;   // blocks up to it hide no key
    const int nblk = (kb - ka + kBlk - 1) / kBlk;
    const int k0 = ka + (nblk * wave / 4) * kBlk;
    const int e1 = ka + (nblk * (wave + 1) / 4) * kBlk;
    const int k1 = e1 < kb ? e1 : kb;
    u32x4 kr[LD], vr[LD];
    float4 kq[4], vq[4];   // scales of the lane's keys
    auto lookup = [&](int kt) {
      return kt < k1 ? page_block(p.table, p.width, b, kt >> 5, p.bpp, p.num_pages, p.Hkv, u.h, BE) : -2;
    };
    auto load = [&](long long at) {
      const size_t o = (size_t)(at < 0 ? 0 : at);
#pragma unroll
      for (int i = 0; i < LD; ++i) kr[i] = ld_nt(p.k_pages + o * (BITS / 8) + (size_t)(i * 64 + lane) * 16);
#pragma unroll
      for (int i = 0; i < LD; ++i) vr[i] = ld_nt(p.v_pages + o * (BITS / 8) + (size_t)(i * 64 + lane) * 16);
      if constexpr (BITS == 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kq[j] = *reinterpret_cast<const float4*>(p.k_scales + o / D + 8 * j + 4 * h2);
          vq[j] = *reinterpret_cast<const float4*>(p.v_scales + o / D + 8 * j + 4 * h2);
        }
      }
    };
    if (k0 < k1) {
      long long at = lookup(k0);
      load(at);
      long long nat = lookup(k0 + kBlk);
      for (int kt = k0; kt < k1; kt += kBlk) {
        if (at >= 0) {   // uniform
          if (BITS == 16 && kt + kBlk > u.nk) {
#pragma unroll
            for (int i = 0; i < LD; ++i) vr[i] = cut_tail(vr[i], kt + 16 * (i & 1), h2, u.nk);
          }
          auto kop = [&](int i) {
            if constexpr (BITS == 16) return __builtin_bit_cast(bf16x8, kr[i]);
            else
              return __builtin_bit_cast(bf16x8, (i & 1) ? widen8(kr[i >> 1].z, kr[i >> 1].w)
                                                        : widen8(kr[i >> 1].x, kr[i >> 1].y));
          };
          auto vop = [&](int t, int jj) {
            if constexpr (BITS == 16) return vr[2 * t + jj];
            else return jj ? widen8(vr[t].z, vr[t].w) : widen8(vr[t].x, vr[t].y);
          };
          auto part = [](const float4& f, int e) { return e == 0 ? f.x : e == 1 ? f.y : e == 2 ? f.z : f.w; };
          auto ks = [&](int r) { return part(kq[r >> 2], r & 3) * p.scale_log2; };
          auto vs = [&](int r) { return part(vq[r >> 2], r & 3); };
          if (kt + 31 <= wmin)
            attend<D, BITS, 1, false>(s, kt, h2, p.scale_log2, kop, vop, ks, vs);
          else
            attend<D, BITS, 1, true>(s, kt, h2, p.scale_log2, kop, vop, ks, vs);
        } else if (p.status && lane == 0) {
          atomicOr(p.status, kStatusPage);
        }
        if (kt + kBlk < k1) {
          at = nat;
          load(at);
          nat = lookup(kt + 2 * kBlk);
        }
      }
    }
    // The waves' parts, in wave order.
    const float l = s.l[0] + __shfl_xor(s.l[0], 32, 64);
    __syncthreads();   // the previous piece's reads are done
    if (h2 == 0) {
      s_m[wave][c32] = s.m[0];
      s_l[wave][c32] = l;
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(&s_o[wave][c32 * OS + 32 * t + 8 * j + 4 * h2]) =
            make_float4(s.o[0][t][4 * j], s.o[0][t][4 * j + 1], s.o[0][t][4 * j + 2], s.o[0][t][4 * j + 3]);
    __syncthreads();
    const int slot = 2 * g + (starts ? 1 : 0);
    const bool whole = starts && ends;
    if (!whole && ka >= kb) continue;
    for (int idx = 4 * tid; idx < rows * D; idx += 4 * kPT) {
      const int r = idx / D, d = idx % D;
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
        const float inv = ls == 0.f ? 0.f : 1.f / ls;
        store4(out_row(p, rq, u, r) + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * RT + r) * D + d) = v;
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

// Workgroup (g, y): rows [y RB, y RB + RB) of the tile that workgroup g began
// and others finished.
template <int D, int RT, int RB>
__global__ __launch_bounds__(kPT) void attn_join_kernel(PAttn p, int step) {
  const int tid = threadIdx.x, lane = tid & 63;
  const Shares sh(line_total(p, lane), p.G, p.min_share);
  const int g = blockIdx.x;
  if (sh.W == 0 || g + 1 >= sh.G) return;
  const long long hi = sh.lo(g + 1);   // the tile that crosses this line position
  Req rq;
  find_req(p, lane, hi, rq);
  const Tile u = tile_at(p, rq, hi);
  if (u.begin >= hi || u.begin < sh.lo(g)) return;   // none, or begun before g
  const int gl = sh.owner(u.begin + u.len - 1);
  const int rows = u.n * p.rep;
  const int r0 = blockIdx.y * RB;
  if (r0 >= rows) return;
  const int r1 = r0 + RB < rows ? r0 + RB : rows;
  for (int idx = 4 * tid; idx < (r1 - r0) * D; idx += 4 * kPT) {
    const int r = r0 + idx / D, d = idx % D;
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = g; w <= gl; ++w) {
      const long long a = w == g ? 0 : sh.lo(w) - u.begin;
      const int ka = key_at(u, a, step), kb = key_at(u, sh.lo(w + 1) - u.begin, step);
      if (ka >= kb) continue;   // an empty piece left nothing
      const size_t row = (size_t)(2 * w + (w == g ? 1 : 0)) * RT + r;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + row * 2);
      if (ml.x == -INFINITY) {   // no finite score yet: l is 0 or NaN
        l += ml.y;
        continue;
      }
      const float4 a4 = *reinterpret_cast<const float4*>(p.part_o + row * D + d);
      const float mn = fmaxf(m, ml.x);
      const float cm = m == -INFINITY ? 0.f : exp2_fast(m - mn), cw = exp2_fast(ml.x - mn);
      m = mn;
      l = l * cm + ml.y * cw;
      v.x = v.x * cm + a4.x * cw;
      v.y = v.y * cm + a4.y * cw;
      v.z = v.z * cm + a4.z * cw;
      v.w = v.w * cm + a4.w * cw;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store4(out_row(p, rq, u, r) + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  }
}

// Which kernel runs, and its tiles: calls of at most 32 query rows per kv head
// and request (decode, verify) split each piece's keys over the waves and read
// them straight into registers; others share K and V tiles through LDS.
struct AttnPlan {
  bool few;
  int RT, P, G, min_share, step;
};
inline AttnPlan attn_plan(int Hq, int Hkv, int D, int max_rows) {
  const int rep = Hq / Hkv;
  AttnPlan a;
  a.few = max_rows > 0 && (long long)max_rows * rep <= 32;
  a.RT = a.few ? 32 : D == 256 ? 128 : 256;
  a.P = a.RT / rep;
  a.step = a.few ? kBlk : kStepKeys;
  a.G = device_cus();
  a.min_share = a.few ? 4 * kBlk : 2 * kStepKeys;
  return a;
}

template <int D, int BITS>
int launch_attn(const PAttn& p, const AttnPlan& a, hipStream_t st) {
  constexpr int NB = D == 256 ? 1 : 2;
  if (a.few)
    hipLaunchKernelGGL((attn_few_kernel<D, BITS>), dim3((unsigned)p.G), dim3(kPT), 0, st, p);
  else
    hipLaunchKernelGGL((attn_chunk_kernel<D, BITS, NB>), dim3((unsigned)p.G), dim3(kPT), 0, st, p);
  const int rc = launch_check("mtp_paged_attn");
  if (rc) return rc;
  if (a.few)
    hipLaunchKernelGGL((attn_join_kernel<D, 32, 8>), dim3((unsigned)p.G, 4), dim3(kPT), 0, st, p, a.step);
  else
    hipLaunchKernelGGL((attn_join_kernel<D, 128 * NB, 16>), dim3((unsigned)p.G, 8 * NB), dim3(kPT), 0, st, p, a.step);
  return launch_check("mtp_paged_attn");
}

}  // namespace mtp

using namespace mtp;

MTP_API size_t mtp_paged_attn_workspace_bytes(int Hq, int Hkv, int D, int max_rows) {
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 1) return 0;
  const AttnPlan a = attn_plan(Hq, Hkv, D, max_rows);
  return (size_t)2 * a.G * a.RT * (D + 2) * sizeof(float);
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
  p.T = a->T;
  p.B = a->B;
  p.width = a->width;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.rep = a->Hq / a->Hkv;
  p.bpp = a->page_size / kBlk;
  p.num_pages = a->num_pages;
  p.P = plan.P;
  p.G = plan.G;
  p.min_share = plan.min_share;
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
