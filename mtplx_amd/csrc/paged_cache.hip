// Rotary positions of packed tokens, and the paged KV cache's writes (rotating
// and quantising on the way) and reads. All of them move bytes once.
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
    rot_item(it, s.src + (t0 + t) * s.st + hh * s.sh, r.dims, r.trad, cs + t * half,
             [&](int d, uint4 v) { *reinterpret_cast<uint4*>(dst + d) = v; });
  }
}

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

__device__ __forceinline__ long long floor_blk(long long p) { return p >= 0 ? p / kBlk : -((-p + kBlk - 1) / kBlk); }

// Blocks of 32 positions that request b's new tokens fall into, from the
// block of the first one on.
__device__ __forceinline__ int touched_blocks(long long start, int n) {
  return n > 0 ? (int)(floor_blk(start + n - 1) - floor_blk(start)) + 1 : 0;
}

// The request and block that write unit u is, and the number of units in all.
// With row offsets every wave scans the requests' block counts, 64 at a time.
__device__ __forceinline__ bool find_unit(const WriteParams& p, long long u, int lane, int& b, int& blk,
                                          long long& total) {
  if (!p.row_off) {
    total = (long long)p.B * p.nb_uniform;
    b = (int)(u / p.nb_uniform);
    blk = (int)(u % p.nb_uniform);
    return u < total;
  }
  long long carry = 0;
  bool found = false;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int bb = b0 + lane;
    int cnt = 0;
    if (bb < p.B) cnt = touched_blocks(p.q_start[bb], req_rows(p.row_off, bb, p.B, p.T).n);
    int incl = cnt;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(incl, off, 64);
      if (lane >= off) incl += t;
    }
    const bool mine = !found && u >= carry + incl - cnt && u < carry + incl;
    const unsigned long long m = __ballot(mine);
    if (m) {
      const int src = __ffsll((long long)m) - 1;
      b = b0 + src;
      blk = (int)(u - carry) - __shfl(incl - cnt, src, 64);
      found = true;
    }
    carry += __shfl(incl, 63, 64);
  }
  total = carry;
  b = __builtin_amdgcn_readfirstlane(b);
  blk = __builtin_amdgcn_readfirstlane(blk);
  return found;
}

// One unit: a block of 32 positions of one request, one head, K or V. The new
// rows in it go through LDS (K rotated, rounded to bf16 as the standalone
// rotation rounds) and out in the page's order, whole 16-byte chunks wherever
// all their keys are new.
template <int D, int BITS>
__device__ __forceinline__ void write_unit(const WriteParams& p, int b, int blk, int h, bool isk, unsigned char* lds) {
  constexpr int RS = D + 8;   // LDS row: 16-byte reads of 8 rows hit distinct banks
  uint16_t* rows = reinterpret_cast<uint16_t*>(lds);                 // [32][RS]
  float2* cs = reinterpret_cast<float2*>(lds + 32 * RS * 2);         // [32][dims / 2]
  float* sc = reinterpret_cast<float*>(lds + 32 * RS * 2 + 32 * (D / 2) * 8);   // [32] inverse scales
  const int tid = threadIdx.x;
  const ReqRows rq = req_rows(p.row_off, b, p.B, p.T);
  const long long start = p.q_start[b];
  const long long ablk = floor_blk(start) + blk, base = ablk * kBlk;
  // Keys [klo, khi) of the block are new; token of key kk: first + kk.
  const int klo = start > base ? (int)(start - base) : 0;
  const long long end = start + rq.n - base;
  const int khi = end < kBlk ? (int)end : kBlk;
  if (klo >= khi) return;   // uniform (a request of no rows)
  const long long first = rq.lo + (base - start);
  const long long at = page_block(p.block_table, p.width, b, ablk, p.bpp, p.num_pages, p.Hkv, h, kBlk * D);
  if (at < 0) {
    if (p.status && tid == 0) atomicOr(p.status, kStatusPage);
    return;
  }
  const int half = p.r.dims / 2, n = khi - klo;
  if (isk && half) {
    for (int x = tid; x < n * half; x += kNT)
      cs[x] = rot_angle(base + klo + x / half, p.r.table[x % half], p.r.gain);
    __syncthreads();
  }
  const uint16_t* src = isk ? p.k + h * p.k_head : p.v + h * p.v_head;
  const long long st = isk ? p.k_token : p.v_token;
  if (isk && half) {
    const int ipr = rot_items(D, p.r.dims, p.r.trad);
    for (int x = tid; x < n * ipr; x += kNT) {
      const int kk = x / ipr;
      uint16_t* dst = rows + (klo + kk) * RS;
      rot_item(x % ipr, src + (first + klo + kk) * st, p.r.dims, p.r.trad, cs + kk * half,
               [&](int d, uint4 v) { *reinterpret_cast<uint4*>(dst + d) = v; });
    }
  } else {
    for (int x = tid; x < n * (D / 8); x += kNT) {
      const int kk = klo + x / (D / 8), d = (x % (D / 8)) * 8;
      *reinterpret_cast<uint4*>(rows + kk * RS + d) = *reinterpret_cast<const uint4*>(src + (first + kk) * st + d);
    }
  }
  __syncthreads();
  unsigned char* pool = isk ? p.k_pages : p.v_pages;
  if constexpr (BITS == 8) {
    // Eight lanes a row: its largest magnitude, then 127 / A and A / 127 (one
    // correctly rounded division each). A row with a NaN or an infinity gets a
    // NaN scale, so it reads as NaN instead of as wrong numbers; one below
    // 2^-100 gets zeros (127 / A would overflow, A / 127 go subnormal).
    const int kk = tid >> 3, part = tid & 7;
    float a = 0.f;
    bool bad = false;
    if (kk >= klo && kk < khi) {
#pragma unroll
      for (int e = 0; e < D / 8; e += 8) {
        const Chunk8 c = unpack8(*reinterpret_cast<const uint4*>(rows + kk * RS + part * (D / 8) + e));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a = fmaxf(a, fabsf(c.v[i]));
          bad |= !(fabsf(c.v[i]) <= 3.4e38f);
        }
      }
    }
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
      a = fmaxf(a, __shfl_xor(a, off, 64));
      bad |= (bool)__shfl_xor((int)bad, off, 64);
    }
    if (part == 0 && kk >= klo && kk < khi) {
      const bool tiny = a < 0x1p-100f;
      sc[kk] = bad || tiny ? 0.f : 127.f / a;
      float* scales = (isk ? p.k_scales : p.v_scales) + at / D;   // [page][head][slot]
      scales[kk] = bad ? __uint_as_float(0x7fc00000u) : tiny ? 0.f : a / 127.f;
    }
    __syncthreads();
  }
  auto quant = [&](float x, float inv) -> uint32_t {
    // inv = 0 for a row of NaN scale: NaN and inf * 0 count as 0.
    const float q = rintf(__fmul_rn(x, inv));
    return (uint32_t)(q >= -127.f && q <= 127.f ? (int)q : q > 127.f ? 127 : q < -127.f ? -127 : 0) & 0xffu;
  };
  if (isk) {
    constexpr int CH = BITS == 8 ? 16 : 8;
    for (int x = tid; x < 32 * (D / CH); x += kNT) {   // chunk x: key x % 32, the order of the page
      const int kk = x & 31, ih = x >> 5;
      if (kk < klo || kk >= khi) continue;
      const int d = (ih & 1) * (D / 2) + (ih >> 1) * CH;
      const uint16_t* row = rows + kk * RS + d;
      uint4 o;
      if constexpr (BITS == 16) {
        o = *reinterpret_cast<const uint4*>(row);
      } else {
        const float inv = sc[kk];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Chunk8 c = unpack8(*reinterpret_cast<const uint4*>(row + 8 * j));
#pragma unroll
          for (int i = 0; i < 2; ++i)
            w[2 * j + i] = quant(c.v[4 * i], inv) | quant(c.v[4 * i + 1], inv) << 8 |
                           quant(c.v[4 * i + 2], inv) << 16 | quant(c.v[4 * i + 3], inv) << 24;
        }
        o = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(pool + (size_t)at * (BITS / 8) + (size_t)x * 16) = o;
    }
  } else {
    constexpr int JJ = BITS == 8 ? 1 : 2;   // 16-bit chunks hold the keys of one 16, 8-bit chunks of both
    for (int x = tid; x < JJ * D * 2; x += kNT) {
      const int c = x & 31, h2 = (x >> 5) & 1, tj = x >> 6;
      const int d = 32 * (tj / JJ) + c;
      unsigned char* dst = pool + (size_t)at * (BITS / 8) + (size_t)x * 16;
      if constexpr (BITS == 16) {
        const int k16 = 16 * (tj & 1);
        uint16_t e[8];
        bool all = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int kk = k16 + v_slot_key(h2, i);
          const bool in = kk >= klo && kk < khi;
          all &= in;
          e[i] = in ? rows[kk * RS + d] : 0;
        }
        if (all) {
          *reinterpret_cast<uint4*>(dst) = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
                                                      e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int kk = k16 + v_slot_key(h2, i);
            if (kk >= klo && kk < khi) reinterpret_cast<uint16_t*>(dst)[i] = e[i];
          }
        }
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
        bool all = true;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int kk = 16 * (i >> 3) + v_slot_key(h2, i & 7);
          const bool in = kk >= klo && kk < khi;
          all &= in;
          if (in) w[i >> 2] |= quant(bf2f(rows[kk * RS + d]), sc[kk]) << (8 * (i & 3));
        }
        if (all) {
          *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int kk = 16 * (i >> 3) + v_slot_key(h2, i & 7);
            if (kk >= klo && kk < khi) dst[i] = (unsigned char)(w[i >> 2] >> (8 * (i & 3)));
          }
        }
      }
    }
  }
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
constexpr size_t write_lds_bytes() {
  return (size_t)32 * (D + 8) * 2 + (size_t)32 * (D / 2) * 8 + 32 * 4;
}

template <int D, int BITS>
__global__ __launch_bounds__(kNT) void paged_write_kernel(WriteParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[write_lds_bytes<D, BITS>()];
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x >= p.kv_groups) {   // rotate queries, q_tokens at a time
    float2* cs = reinterpret_cast<float2*>(lds);
    __shared__ int s_live[kRotTokens];
    const int half = p.r.dims / 2, ipr = rot_items(D, p.r.dims, p.r.trad);
    const int stride = ((int)gridDim.x - p.kv_groups) * p.q_tokens;
    for (int t0 = ((int)blockIdx.x - p.kv_groups) * p.q_tokens; t0 < p.T; t0 += stride) {
      const int n = p.T - t0 < p.q_tokens ? p.T - t0 : p.q_tokens;
      for (int t = 0; t < n; ++t) {
        long long pos = 0;
        const int b = token_request(p, t0 + t, &pos);   // the same in every thread
        if (threadIdx.x == 0) s_live[t] = b >= 0;
        for (int x = threadIdx.x; x < half; x += kNT) cs[t * half + x] = rot_angle(pos, p.r.table[x], p.r.gain);
      }
      __syncthreads();
      for (int x = threadIdx.x; x < n * p.Hq * ipr; x += kNT) {
        const int it = x % ipr, th = x / ipr;
        const int h = th % p.Hq, t = th / p.Hq;
        if (!s_live[t]) continue;   // rows behind the last request stay as they are
        uint16_t* dst = p.q.dst + (t0 + t) * p.q.dt + h * p.q.dh;
        rot_item(it, p.q.src + (t0 + t) * p.q.st + h * p.q.sh, p.r.dims, p.r.trad, cs + t * half,
                 [&](int d, uint4 v) { *reinterpret_cast<uint4*>(dst + d) = v; });
      }
      __syncthreads();
      if (t0 > p.T - stride) break;   // (t0 + stride could pass 2^31)
    }
    return;
  }
  const long long per = 2LL * p.Hkv;
  for (long long x = blockIdx.x;; x += p.kv_groups) {
    int b = 0, blk = 0;
    long long total = 0;
    if (!find_unit(p, x / per, lane, b, blk, total)) return;   // the same in every thread
    const int hk = (int)(x % per);
    write_unit<D, BITS>(p, b, blk, hk >> 1, (hk & 1) == 0, lds);
    __syncthreads();
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

// One workgroup: a block of 32 positions of one request, one head, K or V,
// back into rows [B, Hkv, count, D].
template <int D, int BITS>
__global__ __launch_bounds__(kNT) void paged_read_kernel(ReadParams p) {
  constexpr int RS = D + 8;
  __shared__ __attribute__((aligned(16))) uint16_t rows[32 * RS];
  __shared__ float sc[32];
  const int tid = threadIdx.x;
  const long long units = 2LL * p.B * p.Hkv * p.nb;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const bool isk = (u & 1) == 0;
    const long long v = u >> 1;
    const int blk = (int)(v % p.nb);
    const int h = (int)(v / p.nb % p.Hkv);
    const int b = (int)(v / p.nb / p.Hkv);
    const long long start = p.start ? p.start[b] : 0;
    const long long ablk = floor_blk(start) + blk, base = ablk * kBlk;
    const int klo = start > base ? (int)(start - base) : 0;
    const long long end = start + p.count - base;
    const int khi = end < kBlk ? (int)end : kBlk;
    if (klo < khi) {   // uniform
      const long long len = p.lengths ? (long long)p.lengths[b] - base : kBlk;
      int live = len < khi ? (len < 0 ? 0 : (int)len) : khi;   // keys [klo, live) are read, [live, khi) are zeros
      if (live < klo) live = klo;
      if (live > klo) {
        const long long at = page_block(p.block_table, p.width, b, ablk, p.bpp, p.num_pages, p.Hkv, h, kBlk * D);
        if (at < 0) {
          if (p.status && tid == 0) atomicOr(p.status, kStatusPage);
          live = klo;
        } else {
          const unsigned char* pool = (isk ? p.k_pages : p.v_pages) + (size_t)at * (BITS / 8);
          if constexpr (BITS == 8) {
            if (tid < 32) sc[tid] = ((isk ? p.k_scales : p.v_scales) + at / D)[tid];
            __syncthreads();
          }
          auto put8 = [&](uint32_t byte, float s) { return f2bf(__fmul_rn((float)(int8_t)byte, s)); };
          constexpr int CH = BITS == 8 ? 16 : 8;
          for (int x = tid; x < 32 * (D / CH); x += kNT) {
            const uint4 c = *reinterpret_cast<const uint4*>(pool + (size_t)x * 16);
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
            if (isk) {
              const int kk = x & 31, ih = x >> 5;
              uint16_t* dst = rows + kk * RS + (ih & 1) * (D / 2) + (ih >> 1) * CH;
              if constexpr (BITS == 16) {
                *reinterpret_cast<uint4*>(dst) = c;
              } else {
                const float s = sc[kk];
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                  *reinterpret_cast<uint32_t*>(dst + i) =
                      put8(w[i >> 2] >> (8 * (i & 3)), s) |
                      (uint32_t)put8(w[i >> 2] >> (8 * (i & 3) + 8), s) << 16;
              }
            } else {
              const int cc = x & 31, h2 = (x >> 5) & 1, tj = x >> 6;
              if constexpr (BITS == 16) {
                const int d = 32 * (tj >> 1) + cc, k16 = 16 * (tj & 1);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  rows[(k16 + v_slot_key(h2, i)) * RS + d] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
              } else {
                const int d = 32 * tj + cc;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const int kk = 16 * (i >> 3) + v_slot_key(h2, i & 7);
                  rows[kk * RS + d] = put8(w[i >> 2] >> (8 * (i & 3)), sc[kk]);
                }
              }
            }
          }
        }
      }
      __syncthreads();
      uint16_t* out = (isk ? p.k_out : p.v_out) + (((size_t)b * p.Hkv + h) * p.count) * D;
      for (int x = tid; x < (khi - klo) * (D / 8); x += kNT) {
        const int kk = klo + x / (D / 8), d = (x % (D / 8)) * 8;
        const size_t j = (size_t)(base + kk - start);
        *reinterpret_cast<uint4*>(out + j * D + d) =
            kk < live ? *reinterpret_cast<const uint4*>(rows + kk * RS + d) : make_uint4(0, 0, 0, 0);
      }
    }
    __syncthreads();
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
  hipLaunchKernelGGL((paged_write_kernel<D, BITS>), dim3((unsigned)groups), dim3(kNT), 0, st, p);
}
template <int D, int BITS>
void launch_read(const ReadParams& p, int groups, hipStream_t st) {
  hipLaunchKernelGGL((paged_read_kernel<D, BITS>), dim3((unsigned)groups), dim3(kNT), 0, st, p);
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
  long long groups = units * 2 * a->Hkv;
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
  long long groups = 2LL * a->B * a->Hkv * p.nb;
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
