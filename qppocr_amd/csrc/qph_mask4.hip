// Attention over the 4-bit cache with first tokens that stay visible or drafted trees
// (kernels: qph_mask4.h): what a call is split into, its checks, and the kernels for
// bfloat16.
#include <algorithm>

#include "qph_mask4.h"

namespace qph {

int launch_mask4_bf16(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s) {
  return launch_mask4<BF16>(g, p, dh, s);
}

static Mask4Plan mask4_plan(const qph_cache4* c, const qph_attn4* p, const qph_attn4_mask* mask) {
  Mask4Plan r{};
  const int64_t rows = std::min<int64_t>((int64_t)p->max_new * (p->heads / c->heads), 1 << 30);
  const int64_t keys = p->window > 0 ? std::min<int64_t>(p->max_len, (int64_t)p->window + p->max_new + 63 +
                                                                         std::min(mask->sinks, kMaxKeys))
                                     : p->max_len;
  const int64_t seqs = (int64_t)p->batch * c->heads;
  r.shared = rows > 32;
  r.nq = rows > 16 ? 2 : 1;
  const int64_t tiles = (rows + mask4_rows(r.nq, r.shared) - 1) / mask4_rows(r.nq, r.shared);
  // (as in attn4_plan: past a million workgroups in all they take further tiles in turn)
  r.row_tiles = (int)std::clamp<int64_t>(tiles, 1, std::max<int64_t>(1, ((int64_t)1 << 20) / seqs));
  r.splits = 1;
  r.chunk = (int64_t)1 << 40;
  const int64_t blocks = r.row_tiles * seqs, most = r.shared ? 1024 : 1536;
  const int64_t least = keys / 512 >= (255 + blocks) / blocks ? 512 : 256;
  if (2 * blocks <= most && keys > 2 * least) {
    int64_t n = std::min<int64_t>({most / blocks, (keys + least - 1) / least, 64});
    r.chunk = ((keys + n - 1) / n + 127) / 128 * 128;
    n = (keys + r.chunk - 1) / r.chunk;
    if (n > 1) r.splits = (int)n;
    else r.chunk = (int64_t)1 << 40;
  }
  if (r.splits > 1) r.workspace = (size_t)r.splits * p->tokens * p->heads * (c->dh + 2) * 4;
  return r;
}

static int mask4_check(const qph_cache4* c, const qph_attn4* p, const qph_attn4_mask* m, int* shift) {
  QPH_TRY(attn4_check(c, p, "attention_mask4", shift));
  if (!m) return fail(QPH_EINVAL, "attention_mask4: NULL arguments");
  if (m->sinks < 0 || m->tree_words < 0) return fail(QPH_EINVAL, "attention_mask4: negative size");
  if (m->tree_words > (1 << 20)) return fail(QPH_EUNSUPPORTED, "attention_mask4: masks of more than 2^20 words");
  if (m->tree_words && m->tree_words < ((int64_t)p->max_new + 63) / 64)
    return fail(QPH_EINVAL, "attention_mask4: masks of " + std::to_string(m->tree_words) +
                                " words for up to " + std::to_string(p->max_new) + " new tokens");
  return QPH_OK;
}

}  // namespace qph

using namespace qph;

extern "C" {

QPH_API int qph_attention_mask4_workspace(const qph_cache4* cache, const qph_attn4* args,
                                          const qph_attn4_mask* mask, size_t* bytes) {
  if (!bytes) return fail(QPH_EINVAL, "attention_mask4_workspace: NULL argument");
  *bytes = 0;
  int shift = 0;
  QPH_TRY(mask4_check(cache, args, mask, &shift));
  if (args->tokens == 0 || args->batch == 0) return QPH_OK;
  *bytes = mask4_plan(cache, args, mask).workspace;
  return QPH_OK;
}

QPH_API int qph_attention_mask4(qph_ctx* ctx, const qph_cache4* cache, const qph_attn4* args,
                                const qph_attn4_mask* mask) {
  int shift = 0;
  QPH_TRY(mask4_check(cache, args, mask, &shift));
  const bool none = args->tokens == 0 || args->batch == 0;
  if (!none && (!args->q || !args->out || !args->lens || (!args->page_table && args->max_pages) ||
                (mask->tree_words && !mask->tree)))
    return fail(QPH_EINVAL, "attention_mask4: NULL argument");
  const Mask4Plan p = none ? Mask4Plan{} : mask4_plan(cache, args, mask);
  if (p.workspace && (!args->workspace || args->workspace_bytes < p.workspace))
    return fail(QPH_EINVAL, "attention_mask4: workspace of " + std::to_string(args->workspace_bytes) +
                                " bytes, needs " + std::to_string(p.workspace));
  if ((uintptr_t)args->workspace % 16)
    return fail(QPH_EINVAL, "attention_mask4: workspace is not 16-byte aligned");
  if ((int64_t)p.row_tiles * p.splits * cache->heads * args->batch > kMaxGroups)
    return fail(QPH_EUNSUPPORTED, "attention_mask4: batch too large for one call");
  if (!ctx) return fail(QPH_EINVAL, "null context");
  if (none) return QPH_OK;
  Mask4 g{};
  g.a = attn4_args(cache, args, shift);
  g.a.row_tiles = p.row_tiles;
  g.a.splits = p.splits;
  g.a.chunk = p.chunk;
  if (p.splits > 1) {
    g.a.part_o = (float*)args->workspace;
    g.a.part_ml = g.a.part_o + (size_t)p.splits * args->tokens * args->heads * cache->dh;
  }
  g.sinks = args->window > 0 ? (int)std::min<int64_t>(mask->sinks, kMaxKeys) : 0;
  g.tree = mask->tree_words ? (const unsigned*)mask->tree : nullptr;
  g.words = 2 * (int)mask->tree_words;
  OnDevice dev(ctx);
  QPH_TRY(dev.rc());
  int rc;
  if (args->dtype == QPH_F32) rc = launch_mask4_f32(g, p, cache->dh, ctx->stream);
  else if (args->dtype == QPH_F16) rc = launch_mask4_f16(g, p, cache->dh, ctx->stream);
  else rc = launch_mask4_bf16(g, p, cache->dh, ctx->stream);
  QPH_TRY(rc);
  return attn4_join(g.a, args->dtype, cache->dh, ctx->stream);
}

}  // extern "C"
