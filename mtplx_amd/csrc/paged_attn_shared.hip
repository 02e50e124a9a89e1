// Attention of a batch whose requests share a long prefix: the kernels of
// paged_attn.hpp over the prefix, once for the rows of all requests, and over
// each request's own keys behind it.
//
// A row's softmax falls into keys [0, P) and [P, its own position]. The first
// part's keys are the same for all requests, so their rows make one list per kv
// head, cut into tiles of 256 (D = 256: 128) as a long chunk's, and K and V of the
// prefix are read once per tile instead of once per request. Every piece of keys
// leaves (o, m, l) of its rows, and so does every piece of a request's own keys;
// the join adds both, m = max m_k, l = sum 2^(m_k - m) l_k, o alike. (The prefix's
// state as the first of a tail's kernel cost 50 us of dependent loads for a wave's
// eight pieces, a join of everything 6.)
//
// What bounds it (40 heads over 8 of 128): 32 requests' four verify rows behind
// 32768 keys, 8 bits: 116 us, of which the prefix 78 (640 rows in tiles of 256:
// 635 TFLOP/s of what there is, 760 with the empty half tile; the chunk kernel's
// 830), the tails 33 (86 MB; 12 us before the first key) and the join 12 (27 MB of
// partials). Without sharing 345. One row of sixteen requests behind 8192 keys, 16
// bits: 40 us (98 without), of 16, 18 and 6.5, each mostly the way of its first loads
// (1 us of the first launch: which request's pages to read).
#include "paged_attn.hpp"

namespace mtp {

template <int D, int BITS>
static int launch_prefix(const char* who, const PAttn& p, int groups, hipStream_t st) {
  hipLaunchKernelGGL((attn_chunk_kernel<D, BITS, kPrefix>), dim3((unsigned)groups), dim3(64 * chunk_waves<D>()), 0, st, p);
  return launch_check(who);
}

int launch_shared(const char* who, PAttn p, const AttnPlan& a, const PrefixPlan& pre, int D, int bits, hipStream_t st) {
  p.prefix_tiles = pre.tiles;
  p.prefix_pieces = pre.pieces;
  p.prefix_rt_log2 = pre.RT == 128 ? 7 : 8;
  PAttn q = p;
  q.rt_log2 = p.prefix_rt_log2;
  q.part_o = const_cast<float*>(p.prefix_o);
  q.part_ml = const_cast<float*>(p.prefix_ml);
  const int groups = (int)((pre.slots(p.Hkv) + 7) / 8 * 8);
  int rc;
  switch (D * 100 + bits) {
    case 6416: rc = launch_prefix<64, 16>(who, q, groups, st); break;
    case 6408: rc = launch_prefix<64, 8>(who, q, groups, st); break;
    case 12816: rc = launch_prefix<128, 16>(who, q, groups, st); break;
    case 12808: rc = launch_prefix<128, 8>(who, q, groups, st); break;
    case 25616: rc = launch_prefix<256, 16>(who, q, groups, st); break;
    default: rc = launch_prefix<256, 8>(who, q, groups, st); break;
  }
  return rc ? rc : launch_scope<kTail>(who, p, a, D, bits, st);
}

}  // namespace mtp
