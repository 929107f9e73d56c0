// dm_kv8_attn.cu — C entries of the attention over the 8-bit paged cache (dm_kv8_attention,
// dm_kv8_attention_workspace): argument checks, the choice of the kernel, the workspace.
#include <cmath>

#include "dm_kv8.h"

namespace dm {

// Workspace: a counter per CTA, two per SM at most (zero between calls), then the partial results.
static size_t counter_bytes(int num_sms) {
    return (static_cast<size_t>(2 * num_sms) * sizeof(unsigned) + 255) / 256 * 256;
}
static size_t workspace_bytes(int D, int num_sms) {
    const size_t k = kv8_keys_part_floats(D, num_sms), q = kv8_queries_part_floats(D, num_sms);
    return counter_bytes(num_sms) + (k > q ? k : q) * sizeof(float);
}

}  // namespace dm

using namespace dm;

extern "C" int32_t dm_kv8_attention_workspace(const dm_kv8_cache* c, uint64_t* bytes, char* eb, uint64_t es) {
    const char* st = "kv8_attention";
    if (eb && es > 0) eb[0] = '\0';
    if (int rc = kv8_check_cache(c, st, eb, es)) return rc;
    if (!bytes) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    Kv8Device g;
    if (int rc = g.enter(c->pages, st, eb, es)) return rc;
    *bytes = workspace_bytes(c->head_dim, g.num_sms);
    return DM_OK;
}

extern "C" int32_t dm_kv8_attention(const dm_kv8_cache* c, const dm_kv8_attn_args* p, void* stream, char* eb,
                                    uint64_t es) {
    const char* st = "kv8_attention";
    if (eb && es > 0) eb[0] = '\0';
    if (int rc = kv8_check_cache(c, st, eb, es)) return rc;
    if (!p) return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null arguments");
    if (p->dtype != DM_DTYPE_BF16 && p->dtype != DM_DTYPE_F32)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "dtype is bf16 or fp32");
    if (p->n < 0 || p->rows < 0 || (p->flags & ~DM_KV8_FILL_ROWS) != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "negative n or rows, or an unknown flag");
    if (p->num_q_heads < 1 || p->num_q_heads % c->num_kv_heads != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "CONFIG_ERROR", st, "num_q_heads %d is no multiple of %d kv heads",
                       p->num_q_heads, c->num_kv_heads);
    if (!std::isfinite(p->sm_scale))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "sm_scale is not finite");
    if (p->table_width < 1 || p->table_width > (1 << 26))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "table_width %d: 1 to 2^26", p->table_width);
    if (p->max_q_len < 1 || (!p->cu_q && (p->max_q_len != 1 || p->rows < p->n)))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st,
                       "need max_q_len >= 1; without cu_q max_q_len is 1 and rows >= n");
    if (static_cast<int64_t>(p->rows) * p->num_q_heads > 0x7fffffffLL)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "rows * num_q_heads must be below 2^31");
    if (p->n == 0 || p->rows == 0) return DM_OK;
    if (!p->q || !p->out || !p->block_table || !p->seq_lens || !p->workspace)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "null pointer");
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0)
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "the workspace must be 256-byte aligned");
    Kv8Device g;
    if (int rc = g.enter(c->pages, st, eb, es)) return rc;
    if (p->workspace_bytes < workspace_bytes(c->head_dim, g.num_sms))
        return kv8_err(eb, es, DM_ERR_INVALID_ARG, "INVALID_ARG", st, "the workspace needs %llu bytes (given %llu)",
                       static_cast<unsigned long long>(workspace_bytes(c->head_dim, g.num_sms)),
                       static_cast<unsigned long long>(p->workspace_bytes));
    Kv8AttnArgs a{};
    a.group = p->num_q_heads / c->num_kv_heads;
    a.pages = c->pages;
    a.scales = c->scales;
    a.q = p->q, a.q_rs = p->q_row_stride, a.q_hs = p->q_head_stride;
    a.out = p->out, a.o_rs = p->out_row_stride, a.o_hs = p->out_head_stride;
    a.lse = p->lse;
    a.table = p->block_table;
    a.seq_lens = p->seq_lens;
    a.cu_q = p->cu_q;
    a.err = kv8_error_word(p->err_dev, g.dev);
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    a.n = p->n;
    a.rows = p->rows;
    a.Hq = p->num_q_heads;
    a.Hkv = c->num_kv_heads;
    a.num_pages = c->num_pages;
    a.width = p->table_width;
    a.max_q = static_cast<int>(p->max_q_len);
    a.fill = (p->flags & DM_KV8_FILL_ROWS) != 0;
    a.counters = static_cast<unsigned*>(p->workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(p->workspace) + counter_bytes(g.num_sms));
    const bool f32 = p->dtype == DM_DTYPE_F32;
    const int elem = f32 ? 4 : 2;
    a.q_vec = kv8_aligned(a.q, a.q_rs, a.q_hs, elem, 32);
    a.o_vec = kv8_aligned(a.out, a.o_rs, a.o_hs, elem, 32);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Many bf16 rows per request and kv head: queries on the M side, 128 rows at a time.  The
    // key-side kernel goes over the cache once per 16 rows but joins small parts; with few items a
    // query-side item is cut into many large ones.  us on the key side / the query side at D = 64
    // and D = 256 (2 kv heads of 8 query heads): 128 items (64 requests of 1000 keys) 32 rows 34/33
    // 52/53, 40 rows 44/33 69/54; 16 items (8 of 4000) 64 rows 31/30 43/48, 96 rows 36/31 51/49; 4 items
    // (2 of 30000) 128 rows 52/51 91/118, 192 rows 68/52 120/115.
    const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
    const int64_t items = (rows + 127) / 128 * a.n * a.Hkv;
    const bool many = !f32 && rows >= (2 * items >= g.num_sms ? 40 : items >= 8 ? 96 : 192);
    const cudaError_t e = many ? launch_kv8_queries(c, a, g.num_sms, g.dev, s)
                               : launch_kv8_keys(c, a, f32, g.num_sms, g.dev, s);
    if (e != cudaSuccess)
        return kv8_err(eb, es, e == cudaErrorInvalidValue ? DM_ERR_INVALID_ARG : DM_ERR_CUDA, "CUDA_ERROR", st,
                       "launch: %s", cudaGetErrorString(e));
    return DM_OK;
}
