// Attention over the paged 4-bit K/V cache: one token per sequence, and runs of tokens.
#include "ttl_kv4.hpp"

#include <cmath>

namespace {

using kv4::Batch;
using kv4::Cache;
using kv4::Layout;

struct Params {
    const float *sinks;
    uint32_t heads, group, window;
    float scale;
};

constexpr uint32_t kThreads = 256;

__device__ inline float as_float(float x) { return x; }
__device__ inline float as_float(__bf16 x) { return float(x); }

// One row and query head a workgroup: 256 positions at a time, a thread per score, then a
// thread per dimension and share of the positions; the running maximum, sum and output of an
// online softmax.
template <int HD, class T>
__global__ __launch_bounds__(kThreads) void attention_kv4_kernel(Cache c, Batch b, Params a, const T *__restrict__ q,
                                                                 T *__restrict__ out) {
    using L = Layout<HD>;
    __shared__ float qs[HD];
    __shared__ float p[kThreads];
    __shared__ uint8_t vscale[kThreads][HD / 32];
    __shared__ const uint8_t *vrecord[kThreads];
    __shared__ float red[kThreads / 64];
    __shared__ uint32_t bad;
    constexpr uint32_t parts = kThreads / HD;
    __shared__ float o_part[parts][HD];
    const uint32_t head = blockIdx.x % a.heads, rown = blockIdx.x / a.heads, t = threadIdx.x;
    const uint32_t kv_head = head / a.group;
    const kv4::Row row = kv4::row_of(b, rown);
    if (row.kind == kv4::kPadding) {
        return;
    }
    T *dst = out + (size_t(rown) * a.heads + head) * HD;
    if (row.kind != kv4::kToken) {
        if (t < HD) {
            dst[t] = T(row.kind == kv4::kIdle ? 0.0f : __builtin_nanf(""));
        }
        return;
    }
    const uint32_t first = a.window && row.position + 1 > a.window ? row.position + 1 - a.window : 0;
    if (t < HD) {
        qs[t] = as_float(q[(size_t(rown) * a.heads + head) * HD + t]);
    }
    if (t == 0) {
        bad = 0;
    }
    __syncthreads();
    if (t < HD && !__builtin_isfinite(qs[t])) {
        bad = 1;
    }
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const uint32_t d = t % HD, part = t / HD;
    for (uint32_t c0 = first; c0 <= row.position; c0 += kThreads) {
        const uint32_t n = min(kThreads, row.position + 1 - c0);
        float s = -INFINITY;
        if (t < n) {
            uint32_t page;
            const uint32_t pos = c0 + t, slot = pos & ((1u << c.page_shift) - 1);
            if (!kv4::page_of(c, b, row.sequence, pos, page)) {
                bad = 1;
                page = 0;
            }
            const uint8_t *rec = kv4::record_of(c, page, kv_head);
            vrecord[t] = rec + L::v_codes(c.page_shift, slot);
            s = 0.0f;
            for (int blk = 0; blk < HD / 32; ++blk) {
                const float sc = kv4::scale_of(rec[L::k_scales(c.page_shift, slot) + blk]);
                vscale[t][blk] = rec[L::v_scales(c.page_shift, slot) + blk];
                for (int w = 0; w < 4; ++w) {
                    float v[8];
                    kv4::values8(*reinterpret_cast<const uint32_t *>(rec + L::k_codes(slot) + blk * 16 + w * 4), sc, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        s = fmaf(qs[blk * 32 + w * 8 + i], v[i], s);
                    }
                }
            }
            s *= a.scale;
        }
        float cm = s;
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) {
            cm = fmaxf(cm, __shfl_xor(cm, x));
        }
        if (t % 64 == 0) {
            red[t / 64] = cm;
        }
        __syncthreads();
        const float m2 = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
        const float base = m2 == -INFINITY ? 0.0f : m2;
        const float x = t < n ? expf(s - base) : 0.0f;
        p[t] = x;
        float sum = x;
#pragma unroll
        for (int y = 32; y >= 1; y >>= 1) {
            sum += __shfl_xor(sum, y);
        }
        __syncthreads();
        if (t % 64 == 0) {
            red[t / 64] = sum;
        }
        __syncthreads();
        const float keep = expf(m - base);
        l = l * keep + ((red[0] + red[1]) + (red[2] + red[3]));
        m = m2;
        o *= keep;
        for (uint32_t i = part; i < n; i += parts) {
            const uint32_t byte = vrecord[i][d / 2];
            float v[8];
            kv4::values8(byte, kv4::scale_of(vscale[i][d / 32]), v);
            o = fmaf(p[i], d % 2 ? v[1] : v[0], o);
        }
        __syncthreads();
    }
    o_part[part][d] = o;
    __syncthreads();
    if (t < HD) {
        float acc = 0.0f;
        for (uint32_t k = 0; k < parts; ++k) {
            acc += o_part[k][t];
        }
        float r;
        if (a.sinks) {
            const float sink = a.sinks[head], top = fmaxf(m, sink);
            r = acc * expf(m - top) / (l * expf(m - top) + expf(sink - top));
        } else {
            r = acc / l;
        }
        dst[t] = T(bad ? __builtin_nanf("") : r);
    }
}

int check_attention(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                    const ttl_kv4_attention *attention, const char *what) {
    TTL_REQUIRE(ctx, TTL_ERR_INVALID, "%s: null context", what);
    const int rc = kv4::check(cache, batch, what);
    if (rc != TTL_OK) {
        return rc;
    }
    TTL_REQUIRE(attention, TTL_ERR_INVALID, "%s: null attention", what);
    const uint32_t heads = attention->heads;
    TTL_REQUIRE(heads >= 1 && heads <= 64 * cache->kv_heads && heads % cache->kv_heads == 0, TTL_ERR_SHAPE,
                "%s: %u heads over %u key/value heads", what, heads, cache->kv_heads);
    TTL_REQUIRE(attention->dtype == TTL_DTYPE_F32 || attention->dtype == TTL_DTYPE_BF16, TTL_ERR_INVALID,
                "%s: type %d is not f32 or bf16", what, attention->dtype);
    TTL_REQUIRE(std::isfinite(attention->scale), TTL_ERR_INVALID, "%s: a scale that is not finite", what);
    return TTL_OK;
}

int run_attention(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                  const ttl_kv4_attention *attention, const void *q, void *out, void *workspace,
                  size_t workspace_bytes, const char *what) {
    const int rc = check_attention(ctx, cache, batch, attention, what);
    if (rc != TTL_OK) {
        return rc;
    }
    if (batch->sequences == 0 || batch->tokens == 0) {
        return TTL_OK;
    }
    TTL_REQUIRE(q && out, TTL_ERR_INVALID, "%s: null argument", what);
    TTL_REQUIRE(((uintptr_t(q) | uintptr_t(out)) & 15) == 0, TTL_ERR_INVALID, "%s: q and out must be 16-byte aligned",
                what);
    const size_t need = ttl_attention_kv4_workspace_bytes(cache, batch, attention);
    TTL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), TTL_ERR_INVALID,
                "%s: a workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : size_t(0), need);
    TTL_REQUIRE(need == 0 || (uintptr_t(workspace) & 255) == 0, TTL_ERR_INVALID,
                "%s: the workspace must be 256-byte aligned", what);
    TTL_REQUIRE(size_t(batch->tokens) * attention->heads <= 0x7fffffffu, TTL_ERR_SHAPE,
                "%s: %u tokens of %u heads are too many for one call", what, batch->tokens, attention->heads);
    TTL_HIP(hipSetDevice(ctx->device));
    const Cache c = kv4::view(cache);
    const Batch b = kv4::view(batch);
    const Params a{attention->sinks, attention->heads, attention->heads / cache->kv_heads, attention->window,
                   attention->scale};
    const uint32_t blocks = b.tokens * a.heads;
    const auto launch = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (attention->dtype == TTL_DTYPE_F32) {
            attention_kv4_kernel<HD, float><<<blocks, kThreads, 0, ctx->stream>>>(
                c, b, a, static_cast<const float *>(q), static_cast<float *>(out));
        } else {
            attention_kv4_kernel<HD, __bf16><<<blocks, kThreads, 0, ctx->stream>>>(
                c, b, a, static_cast<const __bf16 *>(q), static_cast<__bf16 *>(out));
        }
    };
    if (cache->head_dim == 64) {
        launch(std::integral_constant<int, 64>());
    } else {
        launch(std::integral_constant<int, 128>());
    }
    TTL_LAUNCHED(what);
    return TTL_OK;
}

}  // namespace

extern "C" {

size_t ttl_attention_kv4_workspace_bytes(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                                         const ttl_kv4_attention *attention) {
    return 0;
}

int ttl_attention_decode_kv4(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                             const ttl_kv4_attention *attention, const void *q_dev, void *out_dev,
                             void *workspace_dev, size_t workspace_bytes) {
    TTL_REQUIRE(!batch || !batch->starts, TTL_ERR_INVALID,
                "ttl_attention_decode_kv4: takes one token per sequence (starts NULL)");
    return run_attention(ctx, cache, batch, attention, q_dev, out_dev, workspace_dev, workspace_bytes,
                         "ttl_attention_decode_kv4");
}

int ttl_attention_prefill_kv4(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                              const ttl_kv4_attention *attention, const void *q_dev, void *out_dev,
                              void *workspace_dev, size_t workspace_bytes) {
    TTL_REQUIRE(!batch || batch->starts || batch->sequences == 0 || batch->tokens == 0, TTL_ERR_INVALID,
                "ttl_attention_prefill_kv4: null starts");
    return run_attention(ctx, cache, batch, attention, q_dev, out_dev, workspace_dev, workspace_bytes,
                         "ttl_attention_prefill_kv4");
}

}  // extern "C"
