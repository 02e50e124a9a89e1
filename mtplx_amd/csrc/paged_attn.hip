// Attention over the paged KV cache: the entry points, and the kernels of rows
// that see every key up to their own (paged_attn.hpp).
#include "paged_attn.hpp"

using namespace mtp;

MTP_API size_t mtp_paged_attn_workspace_bytes(int Hq, int Hkv, int D, int max_rows) {
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 1) return 0;
  const AttnPlan a = attn_plan(Hq, Hkv, D, max_rows);
  return (size_t)2 * a.G * a.RT * (D + 2) * sizeof(float) + (size_t)a.G * 16;
}

// Whether the prefix is worth a pass of its own: calls of few rows alone (a
// chunk's tile of 256 rows reads K and V once for all of them as it is; tails of
// many rows lost at every prefix but the longest). One tile of rows a request,
// 40 heads over 8, 16 bits, tails of 400: two requests behind 1024 keys 20.6 us
// shared and 19.9 not, behind 2048 20.9 and 22.6; four behind 512 21.0 and 21.8,
// behind 8192 27 and 38; 32 with four rows each behind 1024 40 and 39, behind
// 8192 56 and 113. Several tiles: sixteen requests of eight rows behind 1024 48
// and 36, behind 4096 53 and 61, behind 16384 71 and 161; four of sixteen behind
// 4096 41 and 37, behind 16384 52 and 64.
static bool sharing(const AttnPlan& a, int B, int prefix) {
  if (!a.few || B < 2) return false;
  if (a.tiles == 1) return prefix >= (B < 4 ? 2048 : 1024);
  return prefix >= (B < 8 ? 16384 : 4096);
}

// Whether a windowed call of few rows is dealt (each of its tiles reads the
// window) or takes chunk tiles of 256 rows, of which it fills few: at most two
// tiles always, else up to so many keys in all. 40 heads over 8 of 128, 16 bits:
// sixteen requests of 40 rows a kv head behind 4096 63 us dealt and 67 as chunks
// (8 bits 46 and 71), four of 240 behind 1024 35 and 35, behind 4096 69 and 44 (8
// bits 47 and 51); sixteen of 96, head dim 256, behind 4096 124 and 166.
static bool window_dealt(const AttnPlan& a, int Hkv, int D, int bits, int B, long long keys) {
  if (!a.few || a.tiles <= 2) return a.few;
  return (long long)B * Hkv * a.tiles * keys <= (1LL << 18) * (bits == 8 ? 4 : 1) * (D == 256 ? 4 : 1);
}

MTP_API size_t mtp_paged_attn_scoped_workspace_bytes(int Hq, int Hkv, int D, int max_rows, int T, int B, int shared) {
  const size_t plain = mtp_paged_attn_workspace_bytes(Hq, Hkv, D, max_rows);
  if (!plain || T < 1 || B < 1) return plain;
  const AttnPlan a = attn_plan(Hq, Hkv, D, max_rows, true);
  const int prefix = shared / kBlk * kBlk;
  if (shared > 0)
    return sharing(a, B, prefix) ? scoped_bytes(a, D, B, Hkv, true) + prefix_plan(Hq, Hkv, D, T, prefix).bytes(Hkv, D)
                                 : plain;
  const size_t dealt = scoped_bytes(a, D, B, Hkv, false), chunk = scoped_bytes(attn_plan(Hq, Hkv, D, 0), D, B, Hkv, false);
  return a.few && a.tiles <= 2 ? dealt : dealt > chunk ? dealt : chunk;   // (the keys decide which, else)
}

static int paged_attn(const char* who, const mtp_paged_attn_args* a, const mtp_attn_scope* scope, void* stream) {
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
  AttnPlan plan = attn_plan(a->Hq, a->Hkv, a->D, max_rows, scope != nullptr);
  PrefixPlan pre = {};
  const int prefix = scope ? scope->shared / kBlk * kBlk : 0;
  const long long covered = (long long)a->width * a->page_size;
  if (scope && scope->shared > 0) {
    if (scope->shared > covered) {
      set_error("%s: %d shared positions are more than the table covers", who, scope->shared);
      return MTP_ERR_ARG;
    }
    if (!sharing(plan, a->B, prefix)) {   // each request reads its own keys, as without
      scope = nullptr;
      plan = attn_plan(a->Hq, a->Hkv, a->D, max_rows);
    } else {
      pre = prefix_plan(a->Hq, a->Hkv, a->D, a->T, prefix);
    }
  } else if (scope) {
    const long long keys = (long long)scope->window + scope->sinks;
    if (!window_dealt(plan, a->Hkv, a->D, a->bits, a->B, keys < covered ? keys : covered))
      plan = attn_plan(a->Hq, a->Hkv, a->D, 0);
  }
  if (scope && covered > 0x7fffffffLL - 2 * kBlk) {   // (a block that counts twice would pass 2^31)
    set_error("%s: a table of %lld positions is more than 2^31 - 65", who, covered);
    return MTP_ERR_UNSUPPORTED;
  }
  if (scope && (long long)a->B * a->Hkv > 1 << 20) {
    set_error("%s: %d requests of %d kv heads are more than 2^20", who, a->B, a->Hkv);
    return MTP_ERR_UNSUPPORTED;
  }
  const size_t own = scope ? scoped_bytes(plan, a->D, a->B, a->Hkv, scope->shared > 0)
                           : mtp_paged_attn_workspace_bytes(a->Hq, a->Hkv, a->D, max_rows);
  const size_t need = own + pre.bytes(a->Hkv, a->D);
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
  p.tiles = scope ? plan.tiles : 0;
  p.splits = scope && plan.few ? dealt_splits(plan, a->B, a->Hkv) : 0;
  const size_t slots = p.splits ? dealt_slots(plan, a->B, a->Hkv, scope->shared > 0) : (size_t)2 * plan.G;
  p.part_ml = p.part_o + slots * plan.RT * a->D;
  p.begun = reinterpret_cast<int4*>(p.part_ml + slots * plan.RT * 2);
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
  if (!scope) return launch_scope<kCausal>(who, p, plan, a->D, a->bits, st);
  if (scope->shared > 0) {
    p.shared = scope->shared;
    p.prefix = prefix;
    p.prefix_o = (const float*)((const unsigned char*)a->ws + own);
    p.prefix_ml = p.prefix_o + pre.slots(a->Hkv) * pre.RT * a->D;
    return launch_shared(who, p, plan, pre, a->D, a->bits, st);
  }
  p.window = scope->window;
  p.sinks = scope->sinks;
  // A tile's blocks: the sinks', and those of the window of its first row to its last row.
  p.most = (long long)p.tile_cost + scope->sinks + scope->window + plan.P + 4 * kBlk;
  return launch_window(who, p, plan, a->D, a->bits, st);
}

MTP_API int mtp_paged_attn(const mtp_paged_attn_args* a, void* stream) {
  return paged_attn("mtp_paged_attn", a, nullptr, stream);
}

MTP_API int mtp_paged_attn_scoped(const mtp_paged_attn_args* a, const mtp_attn_scope* scope, void* stream) {
  const char* who = "mtp_paged_attn_scoped";
  if (!scope || scope->window < 0 || scope->sinks < 0 || scope->shared < 0 ||
      (scope->window > 0) == (scope->shared > 0) || (scope->sinks > 0 && !scope->window)) {
    set_error("%s: bad arguments (a window of at least one position, and its sinks, or shared positions)", who);
    return MTP_ERR_ARG;
  }
  return paged_attn(who, a, scope, stream);
}
