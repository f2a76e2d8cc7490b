// C ABI of the multi-axis rotary embedding and of the block-scaled 8-bit cache (include/gtb_attn.h): argument
// checks and the bundles the launchers take.

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <exception>

#include "gtb_common.cuh"
#include "kv8.h"

namespace gtb {
namespace {

bool fail(const char* ctx, const char* what) {
    set_errorf("%s: %s", ctx, what);
    return false;
}

int64_t count(const gtb_tensor4& t) { return t.shape[0] * t.shape[1] * t.shape[2] * t.shape[3]; }

bool is_value_dtype(int dt) { return dt == F32 || dt == F16 || dt == BF16; }

bool contiguous(const gtb_tensor4& t) {
    if (count(t) == 0) return true;
    int64_t s = 1;
    for (int i = 3; i >= 0; --i) {
        if (t.shape[i] > 1 && t.stride[i] != s) return false;
        s *= t.shape[i];
    }
    return true;
}

bool same_shape(const gtb_tensor4& a, const gtb_tensor4& b) {
    for (int i = 0; i < 4; ++i)
        if (a.shape[i] != b.shape[i]) return false;
    return true;
}

bool unit_inner(const gtb_tensor4& t) { return t.shape[3] <= 1 || t.stride[3] == 1; }

Rows3 rows3(const gtb_tensor4& t) { return Rows3{t.data, t.stride[0], t.stride[1], t.stride[2]}; }

bool check_cache(const char* ctx, const gtb_kv8* c) {
    if (!c) return fail(ctx, "the cache is NULL");
    if (c->B < 0 || c->Hkv < 0 || c->Smax < 0 || c->D < 0) return fail(ctx, "negative size");
    if (c->format != GTB_KV8_INT8 && c->format != GTB_KV8_E4M3) return fail(ctx, "the cache must be int8 or e4m3");
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return fail(ctx, "the block of a scale must be 16, 32, 64 or 128 tokens");
    if (c->D < 16 || c->D > 256 || c->D % 16) return fail(ctx, "the head size must be a multiple of 16, at most 256");
    if (c->Smax >= (int64_t)1 << 30) return fail(ctx, "the cache must hold fewer than 2^30 rows a sequence");
    if (c->B > INT32_MAX || c->Hkv > INT32_MAX || c->B * c->Hkv > INT32_MAX)
        return fail(ctx, "batch x kv heads must fit in int32");
    if (c->B == 0 || c->Hkv == 0) return true;
    if (!check_device_ptr(c->lens, ctx, "the cache's lens")) return false;
    if (c->Smax == 0) return true;
    const void* p[4] = {c->k, c->v, c->k_scale, c->v_scale};
    const char* n[4] = {"the cache's k", "the cache's v", "the cache's k_scale", "the cache's v_scale"};
    for (int i = 0; i < 4; ++i)
        if (!check_device_ptr(p[i], ctx, n[i])) return false;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return fail(ctx, "the cache's k and v must be 16-byte aligned");
    return true;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// No C++ exception leaves a C entry point
template <typename F>
int guarded(const char* ctx, F&& f) {
    try {
        return f();
    } catch (const std::exception& e) {
        set_errorf("%s: %s", ctx, e.what());
    } catch (...) {
        set_errorf("%s: unknown error", ctx);
    }
    return -1;
}

// axis and frequency of each pair (64 powers: 4 us, so the last one made stays with the thread)
bool make_rope_table(const char* ctx, const int32_t* sections, int n_axes, int flags, float freq_base, float freq_scale,
                int64_t D, RopeAxesTable& t, int& pairs) {
    if (!sections || n_axes < 1 || n_axes > 4) return fail(ctx, "there must be 1 to 4 sections");
    if (flags & ~(GTB_ROPE_INTERLEAVED | GTB_ROPE_PER_AXIS)) return fail(ctx, "unknown flags");
    int64_t P = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0) return fail(ctx, "sections must not be negative");
        P += sections[a];
    }
    if (P < 1 || 2 * P > D || P > ROPE_MAX_PAIRS) {
        set_errorf("%s: the sections must sum to between 1 and half the head dimension %lld (128 at most), got %lld", ctx,
                   (long long)D, (long long)P);
        return false;
    }
    if (!(freq_base > 0.0f) || !std::isfinite(freq_base) || !std::isfinite(freq_scale))
        return fail(ctx, "freq_base must be positive and finite, and freq_scale finite");
    pairs = (int)P;
    const long double log2_base = std::log2((long double)freq_base);
    int used[4] = {};
    int block = 0, left = sections[0];
    for (int i = 0; i < pairs; ++i) {
        int a;
        if (flags & GTB_ROPE_INTERLEAVED) {
            a = i % n_axes;
            if ((int64_t)i >= (int64_t)n_axes * sections[a]) a = 0;
        } else {
            while (left == 0) left = sections[++block];
            a = block;
            --left;
        }
        const long double e = (flags & GTB_ROPE_PER_AXIS) ? (long double)used[a] / std::max(1, sections[a]) : (long double)i / P;
        ++used[a];
        // (base^-e as 2^(-e log2 base): where e log2 base is large, and with it its rounding, the power is small)
        const long double turns = freq_scale * std::exp2(-e * log2_base) / 6.283185307179586476925286766559005768L;
        // the fraction of a turn per position, rounded to 2^-64; whole turns per position drop out. A position multiplies the
        // error by up to 2^31, so f64's 53 bits would not do (2^-25 of a turn there)
        static_assert(LDBL_MANT_DIG >= 64, "the fraction takes 64 bits");
        const long double frac = turns - std::floor(turns);
        const long double hi = std::floor(std::ldexp(frac, 32));
        const long double lo = std::nearbyint(std::ldexp(std::ldexp(frac, 32) - hi, 32));
        t.turn[i] = ((uint64_t)hi << 32) + (uint64_t)lo;
        t.axis[i] = (uint8_t)a;
    }
    for (int a = 0; a < n_axes; ++a)
        if (used[a] != sections[a])
            return fail(ctx, "interleaved sections must give every axis but the first its turns (n_axes * sections[a] pairs fit)");
    return true;
}

struct RopeKey {
    int32_t sections[4] = {};
    int n_axes = 0, flags = 0;
    float base = 0.0f, scale = 0.0f;
    int64_t D = 0;
    bool operator==(const RopeKey& o) const {
        return std::equal(sections, sections + 4, o.sections) && n_axes == o.n_axes && flags == o.flags && base == o.base &&
               scale == o.scale && D == o.D;
    }
};

}  // namespace

bool rope_table(const char* ctx, const int32_t* sections, int n_axes, int flags, float freq_base, float freq_scale, int64_t D,
                RopeAxesTable& t, int& pairs) {
    thread_local RopeKey last;
    thread_local RopeAxesTable table;
    thread_local int last_pairs;
    thread_local bool made = false;  // `table` is that of `last` (an empty key is a caller's too)
    RopeKey key;
    if (sections && n_axes >= 1 && n_axes <= 4) std::copy(sections, sections + n_axes, key.sections);
    key.n_axes = n_axes;
    key.flags = flags;
    key.base = freq_base;
    key.scale = freq_scale;
    key.D = D;
    if (!made || !(key == last)) {
        made = false;
        if (!make_rope_table(ctx, sections, n_axes, flags, freq_base, freq_scale, D, table, last_pairs)) return false;
        last = key;
        made = true;
    }
    t = table;
    pairs = last_pairs;
    return true;
}

}  // namespace gtb

using namespace gtb;

extern "C" {

GTB_API int gtb_rope_axes(const gtb_tensor4* x, gtb_tensor4* out, const gtb_tensor4* k, gtb_tensor4* k_out,
                          const int32_t* pos, int64_t pos_axis, int64_t pos_batch, const int32_t* sections, int n_axes,
                          int mode, int flags, float freq_base, float freq_scale, int backward, void* stream) {
    const char* ctx = "rope_axes";
    return guarded(ctx, [&]() -> int {
        if (!x || !out || !k != !k_out) return fail(ctx, "x and out, and k and k_out, go together"), -1;
        if (mode != 0 && mode != 2) return fail(ctx, "mode must be 0 (normal) or 2 (NeoX)"), -1;
        RopeAxesArgs a{};
        const gtb_tensor4* in[2] = {x, k};
        const gtb_tensor4* to[2] = {out, k_out};
        for (int w = 0; w < (k ? 2 : 1); ++w) {
            for (int i = 0; i < 4; ++i)
                if (in[w]->shape[i] < 0) return fail(ctx, "negative size"), -1;
            if (!is_value_dtype(in[w]->dtype) || in[w]->dtype != x->dtype) return fail(ctx, "x and k must be f32, f16 or bf16, of one type"), -1;
            if (in[w]->shape[0] != x->shape[0] || in[w]->shape[2] != x->shape[2] || in[w]->shape[3] != x->shape[3])
                return fail(ctx, "x (B, H, S, D) and k (B, Hkv, S, D) do not fit together"), -1;
            if (!same_shape(*in[w], *to[w]) || to[w]->dtype != in[w]->dtype) return fail(ctx, "out must have x's shape and type"), -1;
            if (!unit_inner(*in[w]) || !unit_inner(*to[w])) return fail(ctx, "the innermost stride must be 1"), -1;
            a.x[w] = rows3(*in[w]);
            a.y[w] = rows3(*to[w]);
            a.heads[w] = in[w]->shape[1];
        }
        if (!rope_table(ctx, sections, n_axes, flags, freq_base, freq_scale, x->shape[3], a.tab, a.pairs)) return -1;
        if (x->shape[3] > 256) return fail(ctx, "the head dimension must be at most 256"), -1;
        a.B = x->shape[0];
        a.S = x->shape[2];
        a.D = (int)x->shape[3];
        a.mode = mode;
        a.dtype = x->dtype;
        a.sin_sign = backward ? -1.0f : 1.0f;
        a.pos = pos;
        a.pos_axis = pos_axis;
        a.pos_batch = pos_batch;
        if (a.B == 0 || a.S == 0 || a.heads[0] + a.heads[1] == 0) return 0;
        if (!check_device_ptr(pos, ctx, "positions")) return -1;
        for (int w = 0; w < 2; ++w)
            if (a.heads[w] > 0 && (!check_device_ptr(a.x[w].p, ctx, "x") || !check_device_ptr(a.y[w].p, ctx, "out"))) return -1;
        return launch_rope_axes(a, (cudaStream_t)stream);
    });
}

GTB_API int gtb_kv8_append(const gtb_kv8* cache, const gtb_tensor4* k, const gtb_tensor4* v, const int32_t* counts,
                           int advance, void* stream) {
    const char* ctx = "kv8_append";
    return guarded(ctx, [&]() -> int {
        if (!check_cache(ctx, cache)) return -1;
        if (!k || !v) return fail(ctx, "k and v are required"), -1;
        if (!is_value_dtype(k->dtype) || v->dtype != k->dtype) return fail(ctx, "the new rows must be f32, f16 or bf16, k and v of one type"), -1;
        if (!same_shape(*k, *v) || k->shape[0] != cache->B || k->shape[1] != cache->Hkv || k->shape[3] != cache->D || k->shape[2] < 0) {
            set_errorf("%s: k and v must be (%lld, %lld, n, %lld)", ctx, (long long)cache->B, (long long)cache->Hkv, (long long)cache->D);
            return -1;
        }
        if (k->shape[2] >= (int64_t)1 << 30) return fail(ctx, "fewer than 2^30 rows can be appended at once"), -1;
        if (!unit_inner(*k) || !unit_inner(*v)) return fail(ctx, "the innermost stride of k and v must be 1"), -1;
        if (count(*k) == 0) return 0;
        if (!check_device_ptr(k->data, ctx, "k") || !check_device_ptr(v->data, ctx, "v")) return -1;
        if (counts && !check_device_ptr(counts, ctx, "counts")) return -1;
        int dev = 0;
        if (cuda_failed(cudaGetDevice(&dev), ctx)) return -1;
        int* status = device_status_word(dev);
        if (!status) return fail(ctx, "no status word"), -1;
        return launch_kv8_append(Kv8AppendArgs{*cache, rows3(*k), rows3(*v), k->dtype, k->shape[2], counts, advance, status},
                                 (cudaStream_t)stream);
    });
}

GTB_API int gtb_kv8_read(const gtb_kv8* cache, const int32_t* start, gtb_tensor4* k_out, gtb_tensor4* v_out, void* stream) {
    const char* ctx = "kv8_read";
    return guarded(ctx, [&]() -> int {
        if (!check_cache(ctx, cache)) return -1;
        if (!k_out || !v_out) return fail(ctx, "k_out and v_out are required"), -1;
        if (!is_value_dtype(k_out->dtype) || v_out->dtype != k_out->dtype) return fail(ctx, "the outputs must be f32, f16 or bf16, of one type"), -1;
        if (!same_shape(*k_out, *v_out) || k_out->shape[0] != cache->B || k_out->shape[1] != cache->Hkv ||
            k_out->shape[3] != cache->D || k_out->shape[2] < 0 || !contiguous(*k_out) || !contiguous(*v_out)) {
            set_errorf("%s: the outputs must be contiguous (%lld, %lld, n, %lld)", ctx, (long long)cache->B,
                       (long long)cache->Hkv, (long long)cache->D);
            return -1;
        }
        if (k_out->shape[2] >= (int64_t)1 << 30) return fail(ctx, "fewer than 2^30 rows can be read at once"), -1;
        if (count(*k_out) == 0) return 0;
        if (!check_device_ptr(k_out->data, ctx, "k_out") || !check_device_ptr(v_out->data, ctx, "v_out")) return -1;
        if (((uintptr_t)k_out->data | (uintptr_t)v_out->data) & 15) return fail(ctx, "the outputs must be 16-byte aligned"), -1;
        if (start && !check_device_ptr(start, ctx, "start")) return -1;
        return launch_kv8_read(Kv8ReadArgs{*cache, start, k_out->shape[2], k_out->data, v_out->data, k_out->dtype},
                               (cudaStream_t)stream);
    });
}

GTB_API int gtb_kv8_attention(const gtb_tensor4* q, const gtb_kv8* cache, float scale, const int32_t* counts,
                              const float* score_in, float* score_out, gtb_tensor4* out, float* lse, void* stream) {
    const char* ctx = "kv8_attention";
    return guarded(ctx, [&]() -> int {
        if (!check_cache(ctx, cache)) return -1;
        if (!q || !out) return fail(ctx, "q and out are required"), -1;
        if (!is_value_dtype(q->dtype)) return fail(ctx, "q must be f32, f16 or bf16"), -1;
        for (int i = 0; i < 4; ++i)
            if (q->shape[i] < 0) return fail(ctx, "negative size"), -1;
        if (q->shape[0] != cache->B || q->shape[3] != cache->D) {
            set_errorf("%s: q must be (%lld, H, Lq, %lld)", ctx, (long long)cache->B, (long long)cache->D);
            return -1;
        }
        if (cache->Hkv == 0 || q->shape[1] % cache->Hkv) return fail(ctx, "num_heads must be divisible by num_kv_heads"), -1;
        if (q->shape[1] > INT32_MAX / 2 || q->shape[2] > INT32_MAX / 2 || q->shape[1] / cache->Hkv * q->shape[2] > INT32_MAX / 2)
            return fail(ctx, "too many query rows"), -1;
        if (!same_shape(*q, *out) || out->dtype != q->dtype || !contiguous(*out))
            return fail(ctx, "out must be contiguous, of q's shape and type"), -1;
        if ((uintptr_t)out->data & 15) return fail(ctx, "out must be 16-byte aligned"), -1;
        if (!unit_inner(*q)) return fail(ctx, "the innermost stride of q must be 1"), -1;
        if (!score_in != !score_out) return fail(ctx, "score_in and score_out go together"), -1;
        if (std::isnan(scale) || std::isinf(scale)) return fail(ctx, "scale must be finite"), -1;
        const bool no_rows = count(*q) == 0;
        if (no_rows && (!score_out || score_in == score_out || cache->B == 0)) return 0;
        if (!no_rows && (!check_device_ptr(q->data, ctx, "q") || !check_device_ptr(out->data, ctx, "out"))) return -1;
        if (!no_rows && lse && !check_device_ptr(lse, ctx, "lse")) return -1;
        if (counts && !check_device_ptr(counts, ctx, "counts")) return -1;
        if (score_out && cache->Smax > 0 && cache->B > 0 &&
            (!check_device_ptr(score_in, ctx, "score_in") || !check_device_ptr(score_out, ctx, "score_out")))
            return -1;
        int dev = 0;
        if (cuda_failed(cudaGetDevice(&dev), ctx)) return -1;
        retain_pool_memory(dev);
        gtb_tensor4 o = *out;
        for (int i = 2; i >= 0; --i) o.stride[i] = (i == 2 ? 1 : o.stride[i + 1]) * o.shape[i + 1];
        Kv8AttnArgs a{*cache, rows3(*q), rows3(o), q->dtype, q->shape[1], q->shape[2],
                      scale > 0.0f ? scale : 1.0f / std::sqrt((float)cache->D), counts, score_in, score_out, lse};
        return launch_kv8_attention(a, (cudaStream_t)stream);
    });
}

GTB_API int gtb_kv8_evict(const gtb_kv8* src, const float* score, int64_t budget, int64_t recent, const gtb_kv8* dst,
                          float* score_out, int32_t* kept, void* stream) {
    const char* ctx = "kv8_evict";
    return guarded(ctx, [&]() -> int {
        if (!check_cache(ctx, src) || !check_cache(ctx, dst)) return -1;
        if (dst->B != src->B || dst->Hkv != src->Hkv || dst->D != src->D || dst->format != src->format)
            return fail(ctx, "the two caches must agree in batch, kv heads, head size and format"), -1;
        if (budget < 1 || recent < 0 || recent > budget) {
            set_errorf("%s: budget must be at least 1 and recent between 0 and budget, got %lld and %lld", ctx,
                       (long long)budget, (long long)recent);
            return -1;
        }
        if (dst->Smax < budget) {
            set_errorf("%s: the destination holds %lld rows, fewer than the budget %lld", ctx, (long long)dst->Smax, (long long)budget);
            return -1;
        }
        if (src->B * src->Hkv == 0) return 0;
        if (!check_device_ptr(kept, ctx, "kept")) return -1;
        if (src->Smax > 0 && !check_device_ptr(score, ctx, "score")) return -1;
        if (score_out && !check_device_ptr(score_out, ctx, "score_out")) return -1;
        const int64_t bh = src->B * src->Hkv, ns = bh * src->Smax, nd = bh * dst->Smax;
        const int64_t bs = bh * ((src->Smax + src->block - 1) / src->block), bd = bh * ((dst->Smax + dst->block - 1) / dst->block);
        const void* sp[] = {src->k, src->v, src->k_scale, src->v_scale, src->lens, score};
        const int64_t sn[] = {ns * src->D, ns * src->D, bs * 4, bs * 4, src->B * 4, ns * 4};
        const void* dp[] = {dst->k, dst->v, dst->k_scale, dst->v_scale, dst->lens, score_out, kept};
        const int64_t dn[] = {nd * dst->D, nd * dst->D, bd * 4, bd * 4, dst->B * 4, score_out ? nd * 4 : 0, bh * budget * 4};
        for (int i = 0; i < 6; ++i)
            for (int j = 0; j < 7; ++j)
                if (overlap(sp[i], sn[i], dp[j], dn[j])) return fail(ctx, "source and destination must share no memory"), -1;
        return launch_kv8_evict(Kv8EvictArgs{*src, *dst, score, budget, recent, score_out, kept}, (cudaStream_t)stream);
    });
}

}  // extern "C"
