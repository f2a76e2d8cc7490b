// C ABI of latent attention (include/gtb_attn.h): argument checks and the bundles the launchers take.

#include <cmath>
#include <exception>

#include "gtb_common.cuh"
#include "latent.h"
#include "sdpa_args.h"

namespace gtb {
namespace {

bool fail(const char* ctx, const char* what) {
    set_errorf("%s: %s", ctx, what);
    return false;
}

bool check_latent(const char* ctx, const gtb_latent* c) {
    if (!c) return fail(ctx, "the cache is NULL");
    if (c->B < 0 || c->Smax < 0) return fail(ctx, "negative size");
    if (c->dtype != F16 && c->dtype != BF16) return fail(ctx, "the cache must be f16 or bf16");
    if (c->R < 64 || c->R > 512 || c->R % 64) return fail(ctx, "the latent size must be a multiple of 64, at most 512");
    if (c->Dr < 16 || c->Dr > 64 || c->Dr % 16) return fail(ctx, "the rotary size must be a multiple of 16, at most 64");
    if (c->Smax >= (int64_t)1 << 30) return fail(ctx, "the cache must hold fewer than 2^30 rows a sequence");
    if (c->B > INT32_MAX) return fail(ctx, "the batch must fit in int32");
    if (c->B == 0) return true;
    if (!check_device_ptr(c->lens, ctx, "the cache's lens")) return false;
    if (c->Smax == 0) return true;
    if (!check_device_ptr(c->rows, ctx, "the cache's rows")) return false;
    if ((uintptr_t)c->rows & 15) return fail(ctx, "the cache's rows must be 16-byte aligned");
    return true;
}

template <typename F>
int guarded(const char* ctx, F&& f) {  // no C++ exception leaves a C entry point
    try {
        return f();
    } catch (const std::exception& e) {
        set_errorf("%s: %s", ctx, e.what());
    } catch (...) {
        set_errorf("%s: unknown error", ctx);
    }
    return -1;
}

bool unit_inner(const gtb_tensor4& t) { return t.shape[3] <= 1 || t.stride[3] == 1; }

Rows3 rows3(const gtb_tensor4& t) { return Rows3{t.data, t.stride[0], t.stride[1], t.stride[2]}; }

int* status_of(const char* ctx) {
    int dev = 0;
    if (cuda_failed(cudaGetDevice(&dev), ctx)) return nullptr;
    retain_pool_memory(dev);
    int* s = device_status_word(dev);
    if (!s) fail(ctx, "no status word");
    return s;
}

bool tiled(const gtb_tensor4& t) {  // rows start on 16 bytes, as tile loads and vector stores need
    if (!unit_inner(t) || ((uintptr_t)t.data & 15)) return false;
    for (int i = 0; i < 3; ++i)
        if (t.shape[i] > 1 && (t.stride[i] <= 0 || t.stride[i] % 8)) return false;
    return true;
}

bool is_shape(const gtb_tensor4& t, int64_t a, int64_t b, int64_t c, int64_t d) {
    return t.shape[0] == a && t.shape[1] == b && t.shape[2] == c && t.shape[3] == d;
}

// sizes, types and layout of the expanded form's inputs; `empty`: nothing to compute
bool check_sdpa(const char* ctx, const gtb_tensor4* q, const gtb_tensor4* k, const gtb_tensor4* k_rope, const gtb_tensor4* v,
                const int32_t* lens, float scale, LatentSdpaArgs& a, bool& empty) {
    if (!q || !k || !k_rope || !v) return fail(ctx, "q, k, k_rope and v are required");
    for (const gtb_tensor4* t : {q, k, k_rope, v}) {
        for (int i = 0; i < 4; ++i)
            if (t->shape[i] < 0 || t->shape[i] >= (int64_t)1 << 30) return fail(ctx, "sizes must be from 0 to below 2^30");
        if ((t->dtype != F16 && t->dtype != BF16) || t->dtype != q->dtype) return fail(ctx, "q, k, k_rope and v must be f16 or bf16, of one type");
    }
    a.B = q->shape[0];
    a.H = q->shape[1];
    a.L = q->shape[2];
    a.Hkv = k->shape[1];
    a.S = k->shape[2];
    if (k->shape[3] != 64 && k->shape[3] != 128) return fail(ctx, "k must have 64 or 128 values a head");
    a.Dn = (int)k->shape[3];
    if (q->shape[3] < a.Dn + 16 || q->shape[3] > a.Dn + 64 || q->shape[3] % 16)
        return fail(ctx, "the rotary part must have a multiple of 16 values from 16 to 64");
    a.Dr = (int)q->shape[3] - a.Dn;
    if (k->shape[0] != a.B || !is_shape(*k_rope, a.B, 1, a.S, a.Dr) || !is_shape(*v, a.B, a.Hkv, a.S, a.Dn))
        return fail(ctx, "q (B, H, L, Dn + Dr), k (B, Hkv, S, Dn), k_rope (B, 1, S, Dr) and v (B, Hkv, S, Dn) do not fit together");
    if (a.Hkv == 0 ? a.H != 0 : a.H % a.Hkv) return fail(ctx, "num_heads must be divisible by num_kv_heads");
    if (a.B > 65535 || a.H > 65535) return fail(ctx, "at most 65535 sequences and heads");
    if (lens && a.L != a.S) return fail(ctx, "lengths need as many queries as keys");
    if (!(scale > 0.0f && scale < 1e38f)) return fail(ctx, "scale must be positive and below 1e38");
    a.q = *q;
    a.k = *k;
    a.k_rope = *k_rope;
    a.v = *v;
    a.lens = lens;
    a.scale = scale;
    empty = a.B * a.H == 0 || (a.L == 0 && a.S == 0);
    if (empty) return true;
    if (a.L == 0 || a.S == 0) return fail(ctx, "there must be queries and keys");
    const char* names[4] = {"q", "k", "k_rope", "v"};
    const gtb_tensor4* ts[4] = {q, k, k_rope, v};
    for (int i = 0; i < 4; ++i) {
        if (!check_device_ptr(ts[i]->data, ctx, names[i])) return false;
        if (!tiled(*ts[i])) return fail(ctx, "rows must start on 16 bytes, with a unit innermost stride and positive others");
    }
    if (lens && !check_device_ptr(lens, ctx, "seq_lens")) return false;
    a.status = status_of(ctx);
    return a.status != nullptr;
}

bool check_result(const char* ctx, const gtb_tensor4* t, const gtb_tensor4& like, const char* name) {
    if (!t || t->dtype != like.dtype || !is_shape(*t, like.shape[0], like.shape[1], like.shape[2], like.shape[3])) {
        set_errorf("%s: %s has another shape or type than it should", ctx, name);
        return false;
    }
    if (!check_device_ptr(t->data, ctx, name)) return false;
    if (!tiled(*t)) return fail(ctx, "rows must start on 16 bytes, with a unit innermost stride and positive others");
    return true;
}

}  // namespace
}  // namespace gtb

using namespace gtb;

extern "C" {

GTB_API int gtb_latent_append(const gtb_latent* cache, const gtb_tensor4* latent, const gtb_tensor4* k_rope,
                              const int32_t* counts, const int32_t* offset, int rope_mode, float freq_base, float freq_scale,
                              int advance, void* stream) {
    const char* ctx = "latent_append";
    return guarded(ctx, [&]() -> int {
        if (!check_latent(ctx, cache)) return -1;
        if (!latent || !k_rope) return fail(ctx, "latent and k_rope are required"), -1;
        if ((latent->dtype != F32 && latent->dtype != F16 && latent->dtype != BF16) || k_rope->dtype != latent->dtype)
            return fail(ctx, "latent and k_rope must be f32, f16 or bf16, of one type"), -1;
        const int64_t n = latent->shape[2];
        if (latent->shape[0] != cache->B || latent->shape[1] != 1 || latent->shape[3] != cache->R || n < 0 ||
            k_rope->shape[0] != cache->B || k_rope->shape[1] != 1 || k_rope->shape[2] != n || k_rope->shape[3] != cache->Dr) {
            set_errorf("%s: latent must be (%lld, 1, n, %d) and k_rope (%lld, 1, n, %d)", ctx, (long long)cache->B, cache->R,
                       (long long)cache->B, cache->Dr);
            return -1;
        }
        if (n >= (int64_t)1 << 30) return fail(ctx, "fewer than 2^30 rows can be appended at once"), -1;
        if (!unit_inner(*latent) || !unit_inner(*k_rope)) return fail(ctx, "the innermost strides must be 1"), -1;
        if (rope_mode != -1 && rope_mode != 0 && rope_mode != 2)
            return fail(ctx, "rope_mode must be -1 (keys as given), 0 (normal) or 2 (NeoX)"), -1;
        LatentAppendArgs a{*cache, rows3(*latent), rows3(*k_rope), latent->dtype, n, counts, offset};
        a.turns = rope_mode != -1;
        a.mode = rope_mode;
        a.advance = advance;
        if (a.turns) {
            const int32_t sections = cache->Dr / 2;
            int pairs = 0;
            if (!rope_table(ctx, &sections, 1, 0, freq_base, freq_scale, cache->Dr, a.tab, pairs)) return -1;
        }
        if (cache->B == 0 || n == 0) return 0;
        if (!check_device_ptr(latent->data, ctx, "latent") || !check_device_ptr(k_rope->data, ctx, "k_rope")) return -1;
        if (counts && !check_device_ptr(counts, ctx, "counts")) return -1;
        if (offset && !check_device_ptr(offset, ctx, "offset")) return -1;
        a.status = status_of(ctx);
        return a.status ? launch_latent_append(a, (cudaStream_t)stream) : -1;
    });
}

GTB_API int gtb_latent_attention(const gtb_tensor4* q, const gtb_latent* cache, const gtb_latent* prefix, float scale,
                                 const int32_t* counts, gtb_tensor4* out, float* lse, void* stream) {
    const char* ctx = "latent_attention";
    return guarded(ctx, [&]() -> int {
        if (!check_latent(ctx, cache)) return -1;
        if (prefix) {
            if (!check_latent(ctx, prefix)) return -1;
            if (prefix->B != 1 || prefix->R != cache->R || prefix->Dr != cache->Dr || prefix->dtype != cache->dtype)
                return fail(ctx, "the prefix must be a cache of one sequence with the cache's sizes and type"), -1;
        }
        if (!q || !out) return fail(ctx, "q and out are required"), -1;
        for (int i = 0; i < 4; ++i)
            if (q->shape[i] < 0) return fail(ctx, "negative size"), -1;
        const int64_t H = q->shape[1], Lq = q->shape[2];
        if (q->dtype != cache->dtype || q->shape[0] != cache->B || q->shape[3] != cache->R + cache->Dr) {
            set_errorf("%s: q must be (%lld, H, Lq, %d), of the cache's type", ctx, (long long)cache->B, cache->R + cache->Dr);
            return -1;
        }
        if (out->dtype != q->dtype || out->shape[0] != cache->B || out->shape[1] != H || out->shape[2] != Lq ||
            out->shape[3] != cache->R) {
            set_errorf("%s: out must be (%lld, %lld, %lld, %d), of q's type", ctx, (long long)cache->B, (long long)H,
                       (long long)Lq, cache->R);
            return -1;
        }
        if (H > INT32_MAX / 64 || Lq > INT32_MAX / 64 || (H > 0 && Lq > 0 && cache->B > INT32_MAX / 64 / (H * Lq)))
            return fail(ctx, "too many query rows"), -1;
        if (!(scale > 0.0f && scale < 1e38f)) return fail(ctx, "scale must be positive and below 1e38"), -1;
        if (cache->B * H * Lq == 0) return 0;
        int64_t s = 1;
        for (int i = 3; i >= 0; --i) {
            if (out->shape[i] > 1 && out->stride[i] != s) return fail(ctx, "out must be contiguous"), -1;
            s *= out->shape[i];
        }
        if (!check_device_ptr(q->data, ctx, "q") || !check_device_ptr(out->data, ctx, "out")) return -1;
        if (((uintptr_t)q->data | (uintptr_t)out->data) & 15) return fail(ctx, "q and out must be 16-byte aligned"), -1;
        if (!unit_inner(*q)) return fail(ctx, "the innermost stride of q must be 1"), -1;
        for (int i = 0; i < 3; ++i)
            if (q->shape[i] > 1 && (q->stride[i] <= 0 || q->stride[i] % 8))
                return fail(ctx, "the strides of q must be positive multiples of 16 bytes"), -1;
        if (lse && !check_device_ptr(lse, ctx, "lse")) return -1;
        if (counts && !check_device_ptr(counts, ctx, "counts")) return -1;
        LatentAttnArgs a{*cache, gtb_latent{}, rows3(*q), out->data, H, Lq, scale, counts, lse, status_of(ctx)};
        if (prefix && prefix->Smax > 0) a.prefix = *prefix;
        return a.status ? launch_latent_attention(a, (cudaStream_t)stream) : -1;
    });
}

GTB_API int gtb_latent_sdpa_fwd(const gtb_tensor4* q, const gtb_tensor4* k, const gtb_tensor4* k_rope, const gtb_tensor4* v,
                                const int32_t* seq_lens, float scale, int is_causal, gtb_tensor4* out, float* lse, void* stream) {
    const char* ctx = "latent_sdpa";
    return guarded(ctx, [&]() -> int {
        LatentSdpaArgs a{};
        bool empty = false;
        if (!check_sdpa(ctx, q, k, k_rope, v, seq_lens, scale, a, empty)) return -1;
        if (empty) return 0;
        gtb_tensor4 like = *q;
        like.shape[3] = a.Dn;
        if (!check_result(ctx, out, like, "out")) return -1;
        if (lse && !check_device_ptr(lse, ctx, "lse")) return -1;
        a.o = *out;
        a.lse = lse;
        a.causal = is_causal != 0;
        return launch_latent_sdpa_fwd(a, (cudaStream_t)stream);
    });
}

GTB_API int gtb_latent_sdpa_bwd(const gtb_tensor4* grad_out, const gtb_tensor4* q, const gtb_tensor4* k, const gtb_tensor4* k_rope,
                                const gtb_tensor4* v, const gtb_tensor4* out, const float* lse, const int32_t* seq_lens, float scale,
                                int is_causal, gtb_tensor4* dq, gtb_tensor4* dk, gtb_tensor4* dk_rope, gtb_tensor4* dv, void* stream) {
    const char* ctx = "latent_sdpa_bwd";
    return guarded(ctx, [&]() -> int {
        LatentSdpaArgs a{};
        bool empty = false;
        if (!check_sdpa(ctx, q, k, k_rope, v, seq_lens, scale, a, empty)) return -1;
        if (empty && a.B * a.S > 0) return fail(ctx, "there must be heads, queries and keys"), -1;  // (dk, dk_rope and dv have values)
        if (empty) return 0;
        gtb_tensor4 like = *q;
        like.shape[3] = a.Dn;
        if (!check_result(ctx, grad_out, like, "grad_out") || !check_result(ctx, out, like, "out") || !check_result(ctx, dq, *q, "dq") ||
            !check_result(ctx, dk, *k, "dk") || !check_result(ctx, dk_rope, *k_rope, "dk_rope") || !check_result(ctx, dv, *v, "dv"))
            return -1;
        if (!check_device_ptr(lse, ctx, "lse")) return -1;
        a.g = *grad_out;
        a.o = *out;
        a.lse = const_cast<float*>(lse);
        a.causal = is_causal != 0;
        a.dq = *dq;
        a.dk = *dk;
        a.dk_rope = *dk_rope;
        a.dv = *dv;
        return launch_latent_sdpa_bwd(a, (cudaStream_t)stream);
    });
}

}  // extern "C"
