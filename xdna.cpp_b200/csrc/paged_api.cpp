// C entry points of the paged KV cache operators: the checks of their
// arguments.  What the device data holds is checked by the kernels.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/ggml-b200.h"
#include "gemv.cuh"
#include "paged.cuh"

namespace xb {
namespace {

constexpr int64_t kMaxInt = 0x7fffffff;
// Requests of an attention call: every CTA reads all of their lengths, and the
// threads' shares of them are counted in 32 bits.
constexpr int kMaxAttnSeqs = 1 << 24;

size_t type_size(int type) {
    return type == GGML_TYPE_F32 ? 4 : type == GGML_TYPE_F16 || type == GGML_TYPE_BF16 ? 2 : 0;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

#define REFUSE_IF(cond, ...)    \
    do {                        \
        if (cond) {             \
            set_error(__VA_ARGS__); \
            return false;       \
        }                       \
    } while (0)

bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128 || bs == 256; }

// Checks the cache and gives `kv` its strides.
bool check_cache(const char* what, struct b200_kv_cache& kv) {
    REFUSE_IF(kv.type != GGML_TYPE_F16 && kv.type != GGML_TYPE_BF16, "%s: cache type %d is not F16 or BF16", what,
              kv.type);
    REFUSE_IF(kv.head_dim != 64 && kv.head_dim != 96 && kv.head_dim != 128 && kv.head_dim != 256,
              "%s: head_dim %d is not 64, 96, 128 or 256", what, kv.head_dim);
    REFUSE_IF(kv.kv_heads < 1 || kv.kv_heads > 65535, "%s: kv_heads %d", what, kv.kv_heads);
    REFUSE_IF(!block_size_ok(kv.block_size), "%s: block_size %d is not 16, 32, 64, 128 or 256", what, kv.block_size);
    REFUSE_IF(kv.num_blocks < 1 || kv.num_blocks > kMaxInt / kv.block_size, "%s: num_blocks %ld", what,
              long(kv.num_blocks));
    REFUSE_IF(!kv.k || !kv.v || !aligned16(kv.k) || !aligned16(kv.v), "%s: k and v must be 16-byte aligned", what);
    const int64_t row = 2 * kv.head_dim;
    if (!kv.nb_token && !kv.nb_head && !kv.nb_block) {
        kv.nb_token = row;
        kv.nb_head = row * kv.block_size;
        kv.nb_block = kv.nb_head * kv.kv_heads;
    }
    const int64_t most = int64_t(1) << 39;  // a tensor map's limit on a stride is 2^40
    for (int64_t nb : {kv.nb_token, kv.nb_head, kv.nb_block})
        REFUSE_IF(nb < row || nb % 16 || nb > most, "%s: cache stride %ld is not a multiple of 16 in [%ld, 2^39]",
                  what, long(nb), long(row));
    return true;
}

bool check_rows(const char* what, const char* name, const void* ptr, int64_t& nb, int64_t row) {
    if (nb == 0) nb = row;
    REFUSE_IF(!ptr || !aligned16(ptr), "%s: %s must be 16-byte aligned", what, name);
    REFUSE_IF(nb < row || nb % 16, "%s: %s stride %ld is not a multiple of 16 of at least %ld", what, name, long(nb),
              long(row));
    return true;
}

bool check_plan(const struct b200_kv_plan_args& p) {
    const char* what = "b200_kv_plan";
    REFUSE_IF(p.n_seqs < 0 || p.n_seqs > kMaxSeqs, "%s: n_seqs %d is not in 0 .. %d", what, p.n_seqs, kMaxSeqs);
    REFUSE_IF(!block_size_ok(p.block_size), "%s: block_size %d is not 16, 32, 64, 128 or 256", what, p.block_size);
    REFUSE_IF(p.table_width < 0 || p.table_width > kMaxInt || p.n_free < 0 || p.n_free > kMaxInt || p.max_tokens < 0 ||
                  p.max_tokens > kMaxInt,
              "%s: table_width %ld, n_free %ld or max_tokens %ld is not in 0 .. 2^31 - 1", what, long(p.table_width),
              long(p.n_free), long(p.max_tokens));
    REFUSE_IF(!p.cu_new || !p.status || (p.n_seqs && (!p.cached_lens || !p.new_lens || !p.kv_lens)) ||
                  (p.n_seqs && p.table_width && !p.block_table) || (p.n_free && !p.free_blocks) ||
                  (p.max_tokens && !p.slots),
              "%s: null pointer", what);
    return true;
}

bool check_rope(struct b200_qk_norm_rope_args& p, struct b200_kv_cache& kv) {
    const char* what = "b200_qk_norm_rope";
    if (!check_cache(what, kv)) return false;
    const size_t in = type_size(p.in_type), out = type_size(p.out_type);
    REFUSE_IF(!in || !out, "%s: types %d -> %d are not F32, F16 or BF16", what, p.in_type, p.out_type);
    REFUSE_IF(p.n_tokens < 0 || p.n_tokens > kMaxInt, "%s: n_tokens %ld", what, long(p.n_tokens));
    REFUSE_IF(p.heads < 1 || p.heads > 65535, "%s: heads %d", what, p.heads);
    REFUSE_IF(p.n_rot < 0 || p.n_rot > kv.head_dim || p.n_rot % 8, "%s: n_rot %d is not a multiple of 8 in 0 .. %d",
              what, p.n_rot, kv.head_dim);
    REFUSE_IF(p.n_rot && !(p.freq_base > 0.f && std::isfinite(p.freq_base) && std::isfinite(p.freq_scale)),
              "%s: freq_base %g, freq_scale %g", what, p.freq_base, p.freq_scale);
    REFUSE_IF((p.q_norm || p.k_norm) && !(p.eps >= 0.f && std::isfinite(p.eps)), "%s: eps %g", what, p.eps);
    REFUSE_IF(!aligned16(p.q_norm) || !aligned16(p.k_norm), "%s: norm weights must be 16-byte aligned", what);
    if (p.n_tokens == 0) return true;
    REFUSE_IF(!p.positions || !p.slots, "%s: null pointer", what);
    if (!check_rows(what, "q", p.q, p.nb_q, int64_t(p.heads) * kv.head_dim * in) ||
        !check_rows(what, "k", p.k, p.nb_k, int64_t(kv.kv_heads) * kv.head_dim * in) ||
        !check_rows(what, "v", p.v, p.nb_v, int64_t(kv.kv_heads) * kv.head_dim * in) ||
        !check_rows(what, "q_out", p.q_out, p.nb_q_out, int64_t(p.heads) * kv.head_dim * out))
        return false;
    REFUSE_IF(p.q_out == p.q && (p.in_type != p.out_type || (p.n_tokens > 1 && p.nb_q != p.nb_q_out)),
              "%s: q_out is q with another type (%d, %d) or stride (%ld, %ld)", what, p.in_type, p.out_type,
              long(p.nb_q), long(p.nb_q_out));
    return true;
}

bool check_attention(struct b200_paged_attention_args& p, struct b200_kv_cache& kv) {
    const char* what = "b200_paged_attention";
    if (!check_cache(what, kv)) return false;
    REFUSE_IF((p.q_type != GGML_TYPE_F32 && p.q_type != kv.type) || (p.out_type != GGML_TYPE_F32 && p.out_type != kv.type),
              "%s: q type %d and out type %d are not F32 or the cache's (%d)", what, p.q_type, p.out_type, kv.type);
    REFUSE_IF(p.n_tokens < 0 || p.n_seqs < 0 || p.heads < 1 || p.heads % kv.kv_heads || p.heads > 65535 ||
                  p.n_tokens > kMaxInt / p.heads,
              "%s: n_tokens %ld, n_seqs %d, heads %d over kv_heads %d", what, long(p.n_tokens), p.n_seqs, p.heads,
              kv.kv_heads);
    REFUSE_IF(p.n_seqs > kMaxAttnSeqs, "%s: n_seqs %d is not in 0 .. 2^24", what, p.n_seqs);
    REFUSE_IF(p.table_width < 0 || p.table_width > kMaxInt, "%s: table_width %ld", what, long(p.table_width));
    REFUSE_IF(p.max_new < 0 || p.max_kv < 0 || p.window < 0, "%s: max_new %d, max_kv %d or window %d is negative", what,
              p.max_new, p.max_kv, p.window);
    REFUSE_IF(!std::isfinite(p.scale) || !(p.logit_softcap >= 0.f && std::isfinite(p.logit_softcap)) ||
                  !(p.max_bias >= 0.f && std::isfinite(p.max_bias)),
              "%s: scale %g, logit_softcap %g, max_bias %g", what, p.scale, p.logit_softcap, p.max_bias);
    // the score's factor in units of log 2, and (with a cap) that of tanh's exponential
    const float factor = p.logit_softcap != 0.f ? 4.f * (p.scale / p.logit_softcap) : 2.f * p.scale;
    REFUSE_IF(!std::isfinite(factor), "%s: scale %g with logit_softcap %g passes F32's range", what, p.scale,
              p.logit_softcap);
    if (p.n_tokens == 0 || p.n_seqs == 0) return true;
    REFUSE_IF(!p.cu_new || !p.kv_lens || (p.table_width && !p.block_table), "%s: null pointer", what);
    const int64_t row = int64_t(p.heads) * kv.head_dim;
    return check_rows(what, "q", p.q, p.nb_q, row * int64_t(type_size(p.q_type))) &&
           check_rows(what, "out", p.out, p.nb_out, row * int64_t(type_size(p.out_type)));
}

int done(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return 0;
    set_error("%s: %s", what, cudaGetErrorString(e));
    return -1000 - static_cast<int>(e);
}

}  // namespace
}  // namespace xb

using namespace xb;

extern "C" {

int b200_kv_plan(const struct b200_kv_plan_args* plan, void* stream) {
    if (!plan) {
        set_error("b200_kv_plan: null argument record");
        return -1;
    }
    if (!check_plan(*plan)) return -1;
    return done(kv_plan_launch(*plan, static_cast<cudaStream_t>(stream)), "b200_kv_plan");
}

int b200_qk_norm_rope(const struct b200_qk_norm_rope_args* p, const struct b200_kv_cache* kv, void* stream) {
    if (!p || !kv) {
        set_error("b200_qk_norm_rope: null argument record");
        return -1;
    }
    struct b200_qk_norm_rope_args q = *p;
    struct b200_kv_cache c = *kv;
    if (!check_rope(q, c)) return -1;
    if (q.n_tokens == 0) return 0;
    return done(qk_norm_rope_launch(q, c, static_cast<cudaStream_t>(stream)), "b200_qk_norm_rope");
}

size_t b200_paged_attention_workspace(const struct b200_paged_attention_args* p, const struct b200_kv_cache* kv) {
    if (!p || !kv) {
        set_error("b200_paged_attention_workspace: null argument record");
        return 0;
    }
    struct b200_paged_attention_args q = *p;
    struct b200_kv_cache c = *kv;
    if (!check_attention(q, c) || q.n_tokens == 0 || q.n_seqs == 0) return 0;
    return paged_attention_workspace(q, c);
}

int b200_paged_attention(const struct b200_paged_attention_args* p, const struct b200_kv_cache* kv, void* stream) {
    if (!p || !kv) {
        set_error("b200_paged_attention: null argument record");
        return -1;
    }
    struct b200_paged_attention_args q = *p;
    struct b200_kv_cache c = *kv;
    if (!check_attention(q, c)) return -1;
    if (q.n_tokens == 0 || q.n_seqs == 0) return 0;
    const size_t need = paged_attention_workspace(q, c);
    if (need && (q.workspace_bytes < need || !q.workspace || !aligned16(q.workspace))) {
        set_error("b200_paged_attention: needs %zu bytes of 16-byte aligned workspace, got %zu", need,
                  q.workspace_bytes);
        return -1;
    }
    return done(paged_attention_launch(q, c, static_cast<cudaStream_t>(stream)), "b200_paged_attention");
}

int b200_paged_attention_error(int* status) {
    if (!status) {
        set_error("b200_paged_attention_error: null status pointer");
        return -1;
    }
    return done(paged_error_status(status), "b200_paged_attention_error");
}

}  // extern "C"
