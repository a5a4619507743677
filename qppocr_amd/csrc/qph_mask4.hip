// Attention over the 4-bit cache with first tokens that stay visible or drafted trees
// (kernels: qph_mask4.h): what a call is split into, its checks, and the kernels for
// bfloat16.
#include <algorithm>

#include "qph_mask4.h"

namespace qph {

int launch_mask4_bf16(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s) {
  return launch_mask4<BF16>(g, p, dh, s);
}

// Joins the splits of a row: dh / 4 lanes a row, four elements each, as many rows a wave as
// its lanes hold.  A lane takes the splits' maxima and sums one after the other, then their
// elements, eight in flight.
template <typename E>
__global__ __launch_bounds__(256) void mask4_join_kernel(Attn4 a, int dh, int each) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = dh / 4, sub = lane / per, at = lane - sub * per;
  const int qheads = a.heads * a.group;
  const int64_t all = a.tokens * qheads;
  const float c = fabsf(a.scale) * kLog2e;
  for (int64_t row = ((int64_t)blockIdx.x * 4 + wave) * each + sub; row - sub < all;
       row += (int64_t)gridDim.x * 4 * each) {
    const int64_t t = row / qheads;
    if (sub >= each || row >= all) continue;
    if (a.starts && (t < a.starts[0] || t >= a.starts[a.batch])) continue;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; s++) top = fmaxf(top, a.part_ml[2 * (s * all + row)]);
    float sum = 0.0f;
    bool some = false;
    f32x4 v = {0, 0, 0, 0};
    for (int s0 = 0; s0 < a.splits; s0 += 8) {
      f32x4 u[8];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int64_t part = (int64_t)min(s0 + i, a.splits - 1) * all + row;
        const float m = a.part_ml[2 * part], l = a.part_ml[2 * part + 1];
        // (splits without keys have stored nothing)
        const bool there = s0 + i < a.splits && l != 0.0f;
        w[i] = there ? exp2_(rescale(m, top, c)) : 0.0f;
        sum += there ? w[i] * l : 0.0f;
        some |= there;
        u[i] = f32x4{0, 0, 0, 0};
        if (there) u[i] = *(const f32x4*)(a.part_o + part * dh + 4 * at);
      }
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += w[i] * u[i][e];
    }
    if (a.lse && at == 0) a.lse[row] = some ? log_sum(top, sum, fabsf(a.scale)) : -INFINITY;
    const float inv = some ? 1.0f / sum : 0.0f;
    typename E::type y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (typename E::type)(v[e] * inv);
    __builtin_memcpy((typename E::type*)a.out + t * a.ot + (row % qheads) * a.oh + 4 * at, y, sizeof y);
  }
}

template <typename E>
static int launch_mask4_join(const Attn4& a, int dh, hipStream_t s) {
  const int each = 64 / (dh / 4);
  const int64_t rows = a.tokens * a.heads * a.group;
  const dim3 grid((unsigned)std::min<int64_t>((rows + 4 * each - 1) / (4 * each), 1 << 20));
  hipLaunchKernelGGL(mask4_join_kernel<E>, grid, dim3(256), 0, s, a, dh, each);
  return launch_check("mask4_join_kernel");
}

// How a call is split.  Up to two tiles of rows of a sequence and head take the few-row form.
// Up to 256 rows take it too while its workgroups all run at once and read little of the cache
// between them: each decodes the keys of its 32 rows anew, which costs less than the many-row
// form's longer way to its first product.  (bfloat16, 32 query heads over 8; few-row against many-row
// form: one sequence, 256 rows of 130 keys 14 and 22 us, of 4000 keys 32 and 49, of 16000 64
// and 60; eight sequences, 128 rows of 4000 keys 50 and 54; 24 sequences, 96 rows of 1500 keys
// 31 and 48, 256 rows of 130 keys 33 and 24.  float32: eight sequences, 40 rows of 16000 keys
// 88 and 110 us, 128 rows 192 and 158.  Two tiles, heads of 128 and of 64 in float16, of 64 in
// float32: 64 sequences, 64 rows of up to 4000 keys 124 and 147, 87 and 114, 106 and 130; 16
// sequences, 48 rows of up to 16000 keys 101 and 131, 74 and 101, 87 and 119; bfloat16, 32
// sequences, 64 rows of up to 8000 keys 120 and 110, of 96 elements 127 and 105.)
static Mask4Plan mask4_plan(const qph_cache4* c, const qph_attn4* p, const qph_attn4_mask* mask) {
  Mask4Plan r{};
  const int64_t rows = std::min<int64_t>((int64_t)p->max_new * (p->heads / c->heads), 1 << 30);
  const int64_t keys = p->window > 0 ? std::min<int64_t>(p->max_len, (int64_t)p->window + p->max_new + 63 +
                                                                         std::min(mask->sinks, kMaxKeys))
                                     : p->max_len;
  const int64_t seqs = (int64_t)p->batch * c->heads;
  const int terms = p->dtype == QPH_F32 ? 3 : 1, w = c->dh / 32;
  r.nq = rows > 16 ? mask4_nq(terms, w) : 1;
  int64_t tiles = (rows + 16 * r.nq - 1) / (16 * r.nq);
  const bool few = tiles <= 2 || (rows <= 256 && tiles * seqs <= 768 && tiles * seqs * keys <= 1000000);
  if (!few) {
    // (a launch has fewer than 2^32 threads: four waves a workgroup where eight of so many
    // sequences' heads pass that)
    const int64_t most = seqs <= (((int64_t)1 << 32) - 1) / 512 ? mask4_waves(terms, w) : 4;
    const int64_t groups = (tiles + most - 1) / most;
    r.waves = (int)std::max<int64_t>((tiles + groups - 1) / groups, 4);
    tiles = groups;
  }
  // (as in attn4_plan: past a million workgroups in all they take further tiles in turn)
  r.row_tiles = (int)std::clamp<int64_t>(tiles, 1, std::max<int64_t>(1, ((int64_t)1 << 20) / seqs));
  r.splits = 1;
  r.chunk = (int64_t)1 << 40;
  const int64_t blocks = r.row_tiles * seqs;
  // Keys are split until the workgroups fill the chip: three to a CU in the few-row form; in
  // the many-row form one of more than four waves, or of four waves two, and four where
  // sequences of several lengths make some end early.  A split has 512 keys at least, 256
  // where that leaves CUs idle.
  const int64_t most = !r.waves ? 768 : (r.waves > 4 ? 256 : (p->batch > 1 ? 1024 : 512));
  const int64_t least = keys / 512 >= (255 + blocks) / blocks ? 512 : 256;
  int64_t n = 1;
  if (2 * blocks <= most && keys > 2 * least)
    n = std::min<int64_t>({most / blocks, (keys + least - 1) / least, 64});
  // Three splits of few rows where a CU has one workgroup at most: twelve waves of it instead,
  // the same number without the join's launch.  (One token, twelve waves against three splits:
  // 32 sequences of 8 heads, windows of 4096 36.8 and 40.0 us; 25 sequences of 1100 keys, heads
  // of 128 and 32 16.7 and 21.4, 11.0 and 15.0; 8 sequences of 16 heads of 700 keys, bfloat16
  // 13.4 and 15.2, float16 14.8 and 16.4.  In up to 32 workgroups, whose splits have a CU each,
  // heads of 128 lose up to 8 %: one sequence of one head of 700 keys 12.2 and 11.9, float16
  // 13.3 and 12.3; smaller heads gain there too: of 64 10.2 and 10.6, of 32 9.5 and 10.3.)  Two
  // splits are kept: eight waves a workgroup leave some CUs two (40 sequences: 58 us, 47 with
  // splits).
  r.few = !r.waves && r.nq == 1 && n == 3 && blocks <= 256 ? mask4_few_waves<1>(terms, w) : 4;
  if (r.few > 4) n = 1;
  // Several sequences of one row tile each: even shares of all their keys, which the
  // workgroups find from the lengths (each lane one sequence's), in place of splits of as many
  // keys, of which the chip had to wait for the last full ones (trees of 32 tokens, ragged
  // sequences, 8 heads: 32 of up to 8192 keys 135 us, 156 with equal splits; 6 of up to 32000
  // 124, 149; equal lengths: the same).  A sequence has at most twice the parts that all
  // have on average, and two that begin or end inside a share.
  if (n > 1 && r.waves && r.row_tiles == 1 && p->batch > 1 && p->batch <= 64) {
    r.even = 1;
    r.splits = (int)std::min<int64_t>(2 * (r.waves > 4 ? 256 : 512) / blocks + 2, 64);
    n = 1;
  }
  if (n > 1) {
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
  if (((uintptr_t)cache->k_scales | (uintptr_t)cache->v_scales) % 4)
    return fail(QPH_EINVAL, "attention_mask4: scales are not 4-byte aligned");
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
  // Joined by attn4_join where splits are many and rows few (its workgroups share a row's
  // splits), else with several rows a wave.
  if (p.splits == 1) return QPH_OK;
  if (p.splits > 8 && args->tokens * args->heads < 4096)
    return attn4_join(g.a, args->dtype, cache->dh, ctx->stream);
  if (args->dtype == QPH_F32) return launch_mask4_join<F32>(g.a, cache->dh, ctx->stream);
  if (args->dtype == QPH_F16) return launch_mask4_join<F16>(g.a, cache->dh, ctx->stream);
  return launch_mask4_join<BF16>(g.a, cache->dh, ctx->stream);
}

}  // extern "C"
