// The paged 4-bit K/V cache: descriptor checks, the store of new tokens, the read-back.
#include "ttl_kv4.hpp"

namespace kv4 {

int check(const ttl_kv4_cache *cache, const char *what) {
    TTL_REQUIRE(cache && cache->pool, TTL_ERR_INVALID, "%s: null cache or pool", what);
    TTL_REQUIRE(cache->head_dim == 64 || cache->head_dim == 128, TTL_ERR_SHAPE, "%s: head_dim %u is not 64 or 128",
                what, cache->head_dim);
    TTL_REQUIRE(cache->kv_heads >= 1 && cache->kv_heads <= 256, TTL_ERR_SHAPE, "%s: kv_heads %u is not 1..256", what,
                cache->kv_heads);
    const uint32_t p = cache->page_positions;
    TTL_REQUIRE(p >= 16 && p <= 256 && (p & (p - 1)) == 0, TTL_ERR_SHAPE,
                "%s: page_positions %u is not 16, 32, 64, 128 or 256", what, p);
    TTL_REQUIRE(cache->pages >= 1 && cache->pages <= 0x7fffffffu, TTL_ERR_SHAPE, "%s: a pool of %u pages", what,
                cache->pages);
    TTL_REQUIRE((uintptr_t(cache->pool) & 15) == 0, TTL_ERR_INVALID, "%s: the pool must be 16-byte aligned", what);
    return TTL_OK;
}

int check(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, const char *what) {
    const int rc = check(cache, what);
    if (rc != TTL_OK) {
        return rc;
    }
    TTL_REQUIRE(batch, TTL_ERR_INVALID, "%s: null batch", what);
    TTL_REQUIRE(batch->sequences <= 1u << 20 && batch->tokens <= 1u << 24, TTL_ERR_SHAPE,
                "%s: %u sequences, %u tokens (at most 2^20, 2^24)", what, batch->sequences, batch->tokens);
    if (batch->sequences == 0 || batch->tokens == 0) {
        return TTL_OK;  // nothing to do
    }
    TTL_REQUIRE(batch->page_table && batch->lengths, TTL_ERR_INVALID, "%s: null page table or lengths", what);
    TTL_REQUIRE(batch->starts || batch->tokens == batch->sequences, TTL_ERR_SHAPE,
                "%s: %u tokens of %u sequences need their starts", what, batch->tokens, batch->sequences);
    TTL_REQUIRE(batch->max_length >= 1 && batch->max_length <= 1u << 30 &&
                    batch->max_length <= uint64_t(batch->table_stride) * cache->page_positions,
                TTL_ERR_SHAPE, "%s: max_length %u does not fit a page table of %u pages of %u positions", what,
                batch->max_length, batch->table_stride, cache->page_positions);
    return TTL_OK;
}

Cache view(const ttl_kv4_cache *cache) {
    Cache c{};
    c.pool = cache->pool;
    c.kv_heads = cache->kv_heads;
    c.pages = cache->pages;
    c.page_shift = uint32_t(__builtin_ctz(cache->page_positions));
    c.record = cache->head_dim == 64 ? Layout<64>::record(c.page_shift) : Layout<128>::record(c.page_shift);
    return c;
}

Batch view(const ttl_kv4_batch *batch) {
    return {batch->page_table, batch->lengths,      batch->starts,    batch->sequences,
            batch->tokens,     batch->table_stride, batch->max_length};
}

}  // namespace kv4

namespace {

using kv4::Batch;
using kv4::Cache;
using kv4::Layout;

constexpr uint32_t kThreads = 256, kMostGroups = 0xffffffffu / kThreads;  // (a launch's threads are counted in 32 bits)

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

__device__ inline void load4(const float *p, double (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
}
__device__ inline void load4(const __bf16 *p, double (&v)[4]) {
    const bf16x4 x = *reinterpret_cast<const bf16x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = double(float(x[i]));
    }
}
__device__ inline void store4(float *p, const double (&v)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(float(v[0]), float(v[1]), float(v[2]), float(v[3]));
}
// 64 bits to bf16 in one rounding: through an f32 whose last bit is set where bits were
// dropped (round to odd), which no later rounding to 8 bits can mistake for a tie.
__device__ inline __bf16 to_bf16(double x) {
    float f = float(x);
    const double back = double(f);
    if (back != x && x == x) {
        uint32_t u = __float_as_uint(f);
        if (__builtin_fabs(back) > __builtin_fabs(x)) {
            u -= 1;  // towards zero (from infinity: the largest f32)
        }
        f = __uint_as_float(u | 1u);
    }
    return __bf16(f);
}
__device__ inline void store4(__bf16 *p, const double (&v)[4]) {
    *reinterpret_cast<bf16x4 *>(p) = bf16x4{to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
}

// The E2M1 code of magnitude a (of units of the block's scale), nearest, ties to the even
// code, 6 for everything above 5: the number of midpoints below it.
__device__ inline uint32_t e2m1(double a) {
    return uint32_t(a > 0.25) + uint32_t(a >= 0.75) + uint32_t(a > 1.25) + uint32_t(a >= 1.75) + uint32_t(a > 2.5) +
           uint32_t(a >= 3.5) + uint32_t(a > 5.0);
}

// Four values of each of 8 neighbouring lanes (a block of 32) as codes and the block's byte:
// the smallest e with every magnitude below 7 x 2^e is the largest of the lanes' own.
__device__ inline uint32_t quantise(const double (&x)[4], uint32_t &codes) {
    constexpr int kNone = 1 << 20;  // some value is not a finite f32
    double m = 0.0;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m = __builtin_fmax(m, __builtin_fabs(x[i]));
        finite &= __builtin_isfinite(float(x[i]));
    }
    int e2;
    const double f = __builtin_frexp(m, &e2);  // m = f 2^e2, f in [0.5, 1)
    int e = m > 0.0 ? (f < 0.875 ? e2 - 3 : e2 - 2) : -126;
    e = finite ? (e < -126 ? -126 : (e > 125 ? 125 : e)) : kNone;
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        const int other = __shfl_xor(e, d);
        e = e > other ? e : other;
    }
    codes = 0;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t c = e == kNone ? 0u : e2m1(__builtin_ldexp(__builtin_fabs(x[i]), -e));
        any |= c;
        codes |= (e == kNone ? 0u : c | (__builtin_signbit(x[i]) ? 8u : 0u)) << (4 * i);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        any |= __shfl_xor(any, d);
    }
    return e == kNone ? 255u : (any ? uint32_t(e + 127) : 127u);
}

// Bias, rotation and store of new tokens.  HD / 8 lanes take one head of one token: lane j
// dims 4j..4j+3 and, HD / 2 further, the four that they turn with, so a lane's two runs lie
// in two blocks and 8 neighbouring lanes hold a block whole.  Every lane of a workgroup works
// on one token, so its row's sequence, position and page are scalar work.  2308 tokens of 64 and 8
// heads of 64, f32 in, bf16 queries out: 69 MB in 18.0 us, 3.8 TB/s, three quarters of a large
// copy's rate, as a workgroup requests its inputs only when its index entries have arrived (bf16
// in: 45 MB in 16.8 us).  32 tokens take 5.3 us, that chain of dependent loads (starts, lengths,
// page, inputs).
template <int HD, class X, class Q, bool TILED>
__global__ __launch_bounds__(kThreads) void rope_store_kv4_kernel(Cache c, Batch b, uint32_t heads, uint32_t slices,
                                                                  const X *__restrict__ qkv,
                                                                  const float *__restrict__ bias,
                                                                  const float *__restrict__ rope,
                                                                  uint32_t rope_positions, Q *__restrict__ q_out) {
    using L = Layout<HD>;
    constexpr uint32_t lanes = HD / 8;
    const uint32_t token = blockIdx.x / slices;
    kv4::Row row = kv4::row_of(b, token);
    if (row.kind == kv4::kPadding) {
        return;
    }
    uint32_t page = 0;
    if (row.kind == kv4::kToken &&
        (row.position >= rope_positions || !kv4::page_of(c, b, row.sequence, row.position, page))) {
        row.kind = kv4::kBad;
    }
    const uint32_t u = (blockIdx.x % slices) * kThreads + threadIdx.x;
    const uint32_t head = u / lanes, j = u % lanes;
    if (head >= heads + 2 * c.kv_heads) {
        return;  // (whole heads, so the 8 lanes of a block leave together)
    }
    const bool is_q = head < heads, turned = head < heads + c.kv_heads;
    if (row.kind != kv4::kToken) {
        if (is_q) {
            const double fill = row.kind == kv4::kIdle ? 0.0 : __builtin_nan("");
            const double v[4] = {fill, fill, fill, fill};
            Q *dst = q_out + (size_t(token) * heads + head) * HD + 4 * j;
            store4(dst, v);
            store4(dst + HD / 2, v);
        }
        return;
    }
    const size_t width = size_t(heads + 2 * c.kv_heads) * HD;
    const uint32_t col = head * HD + 4 * j;  // in q | k | v
    // tiled: 16 columns hold 8 dims and their 8 partners (v: 16 dims in order)
    const uint32_t at = TILED && turned ? head * HD + (j / 2) * 16 + (j % 2) * 4 : col;
    const uint32_t at2 = TILED && turned ? at + 8 : col + HD / 2;
    const X *in = qkv + size_t(token) * width;
    double lo[4], hi[4];
    load4(in + at, lo);
    load4(in + at2, hi);
    if (bias) {
        double blo[4], bhi[4];
        load4(bias + col, blo);
        load4(bias + col + HD / 2, bhi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] += blo[i];
            hi[i] += bhi[i];
        }
    }
    if (turned) {
        // (cos, sin) of pairs 4j .. 4j + 3
        const float *cs = rope + (size_t(row.position) * (HD / 2) + 4 * j) * 2;
        double c0[4], c1[4];
        load4(cs, c0);
        load4(cs + 4, c1);
        const double co[4] = {c0[0], c0[2], c1[0], c1[2]}, si[4] = {c0[1], c0[3], c1[1], c1[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double x = lo[i], y = hi[i];
            lo[i] = x * co[i] - y * si[i];
            hi[i] = x * si[i] + y * co[i];
        }
    }
    if (is_q) {
        Q *dst = q_out + (size_t(token) * heads + head) * HD + 4 * j;
        store4(dst, lo);
        store4(dst + HD / 2, hi);
        return;
    }
    const uint32_t kv_head = turned ? head - heads : head - heads - c.kv_heads;
    const uint32_t slot = row.position & ((1u << c.page_shift) - 1);
    uint8_t *rec = kv4::record_of(c, page, kv_head);
    uint8_t *codes = rec + (turned ? L::k_codes(slot) : L::v_codes(c.page_shift, slot));
    uint8_t *scales = rec + (turned ? L::k_scales(c.page_shift, slot) : L::v_scales(c.page_shift, slot));
    uint32_t clo, chi;
    const uint32_t slo = quantise(lo, clo), shi = quantise(hi, chi);
    *reinterpret_cast<uint16_t *>(codes + 2 * j) = uint16_t(clo);
    *reinterpret_cast<uint16_t *>(codes + HD / 4 + 2 * j) = uint16_t(chi);
    if (j % 8 == 0) {
        scales[j / 8] = uint8_t(slo);
        scales[HD / 64 + j / 8] = uint8_t(shi);
    }
}

// The cached values of the batch's rows; a thread takes 8 dims of k or v.  Bound by its stores: 16384
// positions of 8 heads of 64 are 76 MB in 18.5 us, 4.1 TB/s; 32 rows take 4.2 us.
template <int HD>
__global__ __launch_bounds__(kThreads) void dequantize_kv4_kernel(Cache c, Batch b, uint32_t slices,
                                                                  float *__restrict__ k_out,
                                                                  float *__restrict__ v_out) {
    using L = Layout<HD>;
    constexpr uint32_t lanes = HD / 8;
    const uint32_t token = blockIdx.x / slices;
    const uint32_t u = (blockIdx.x % slices) * kThreads + threadIdx.x;
    const uint32_t head = u / lanes, j = u % lanes;
    if (head >= 2 * c.kv_heads) {
        return;
    }
    const bool is_k = head < c.kv_heads;
    float *const out = is_k ? k_out : v_out;
    kv4::Row row = kv4::row_of(b, token);
    uint32_t page = 0;
    if (!out || row.kind == kv4::kPadding) {
        return;
    }
    if (row.kind == kv4::kToken && !kv4::page_of(c, b, row.sequence, row.position, page)) {
        row.kind = kv4::kBad;
    }
    const uint32_t kv_head = is_k ? head : head - c.kv_heads;
    float v[8];
    if (row.kind == kv4::kToken) {
        const uint32_t slot = row.position & ((1u << c.page_shift) - 1);
        const uint8_t *rec = kv4::record_of(c, page, kv_head);
        const uint8_t *codes = rec + (is_k ? L::k_codes(slot) : L::v_codes(c.page_shift, slot));
        const uint8_t *scales = rec + (is_k ? L::k_scales(c.page_shift, slot) : L::v_scales(c.page_shift, slot));
        kv4::values8(*reinterpret_cast<const uint32_t *>(codes + 4 * j), kv4::scale_of(scales[j / 4]), v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = row.kind == kv4::kIdle ? 0.0f : __builtin_nanf("");
        }
    }
    float4 *dst = reinterpret_cast<float4 *>(out + (size_t(token) * c.kv_heads + kv_head) * HD + 8 * j);
    dst[0] = make_float4(v[0], v[1], v[2], v[3]);
    dst[1] = make_float4(v[4], v[5], v[6], v[7]);
}

bool aligned16(const void *p) {
    return (uintptr_t(p) & 15) == 0;
}

template <int HD, class X, class Q>
void launch_store(ttl_ctx *ctx, const Cache &c, const Batch &b, uint32_t heads, const void *qkv, bool tiled,
                  const float *bias, const float *rope, uint32_t rope_positions, void *q) {
    const uint32_t slices = ttl::blocks_for(size_t(heads + 2 * c.kv_heads) * (HD / 8), kThreads);
    if (tiled) {
        if constexpr (HD == 64) {
            rope_store_kv4_kernel<HD, X, Q, true><<<b.tokens * slices, kThreads, 0, ctx->stream>>>(
                c, b, heads, slices, static_cast<const X *>(qkv), bias, rope, rope_positions, static_cast<Q *>(q));
        }
        return;
    }
    rope_store_kv4_kernel<HD, X, Q, false><<<b.tokens * slices, kThreads, 0, ctx->stream>>>(
        c, b, heads, slices, static_cast<const X *>(qkv), bias, rope, rope_positions, static_cast<Q *>(q));
}

}  // namespace

extern "C" {

size_t ttl_kv4_pool_bytes(const ttl_kv4_cache *cache) {
    if (!cache) {
        return 0;
    }
    ttl_kv4_cache shape = *cache;
    shape.pool = reinterpret_cast<uint8_t *>(uintptr_t(16));  // the size does not depend on it
    if (kv4::check(&shape, "ttl_kv4_pool_bytes") != TTL_OK) {
        return 0;
    }
    return size_t(cache->pages) * cache->kv_heads * kv4::view(&shape).record;
}

int ttl_qkv_rope_store_kv4(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, uint32_t heads,
                           const void *qkv_dev, int x_dtype, int qkv_order, const float *bias_dev,
                           const float *rope_dev, uint32_t rope_positions, void *q_dev, int q_dtype) {
    TTL_REQUIRE(ctx, TTL_ERR_INVALID, "ttl_qkv_rope_store_kv4: null context");
    const int rc = kv4::check(cache, batch, "ttl_qkv_rope_store_kv4");
    if (rc != TTL_OK) {
        return rc;
    }
    TTL_REQUIRE(heads >= 1 && heads <= 64 * cache->kv_heads && heads % cache->kv_heads == 0, TTL_ERR_SHAPE,
                "ttl_qkv_rope_store_kv4: %u heads over %u key/value heads", heads, cache->kv_heads);
    TTL_REQUIRE((x_dtype == TTL_DTYPE_F32 || x_dtype == TTL_DTYPE_BF16) &&
                    (q_dtype == TTL_DTYPE_F32 || q_dtype == TTL_DTYPE_BF16),
                TTL_ERR_INVALID, "ttl_qkv_rope_store_kv4: types %d and %d are not f32 or bf16", x_dtype, q_dtype);
    TTL_REQUIRE(qkv_order == TTL_QKV_PLAIN || qkv_order == TTL_QKV_TILED, TTL_ERR_INVALID,
                "ttl_qkv_rope_store_kv4: unknown order %d", qkv_order);
    TTL_REQUIRE(qkv_order == TTL_QKV_PLAIN || (heads == 64 && cache->kv_heads == 8 && cache->head_dim == 64),
                TTL_ERR_SHAPE, "ttl_qkv_rope_store_kv4: the tiled order is that of 64 and 8 heads of 64");
    if (batch->sequences == 0 || batch->tokens == 0) {
        return TTL_OK;
    }
    TTL_REQUIRE(qkv_dev && rope_dev && q_dev && rope_positions, TTL_ERR_INVALID,
                "ttl_qkv_rope_store_kv4: null argument");
    TTL_REQUIRE(aligned16(qkv_dev) && aligned16(bias_dev) && aligned16(rope_dev) && aligned16(q_dev), TTL_ERR_INVALID,
                "ttl_qkv_rope_store_kv4: qkv, bias, rope and q must be 16-byte aligned");
    const size_t lanes = size_t(heads + 2 * cache->kv_heads) * (cache->head_dim / 8);
    TTL_REQUIRE(size_t(batch->tokens) * ttl::blocks_for(lanes, kThreads) <= kMostGroups, TTL_ERR_SHAPE,
                "ttl_qkv_rope_store_kv4: %u tokens of %u heads are too many for one call", batch->tokens, heads);
    TTL_HIP(hipSetDevice(ctx->device));
    const Cache c = kv4::view(cache);
    const Batch b = kv4::view(batch);
    const bool tiled = qkv_order == TTL_QKV_TILED;
    const auto launch = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (x_dtype == TTL_DTYPE_F32 && q_dtype == TTL_DTYPE_F32) {
            launch_store<HD, float, float>(ctx, c, b, heads, qkv_dev, tiled, bias_dev, rope_dev, rope_positions, q_dev);
        } else if (x_dtype == TTL_DTYPE_F32) {
            launch_store<HD, float, __bf16>(ctx, c, b, heads, qkv_dev, tiled, bias_dev, rope_dev, rope_positions, q_dev);
        } else if (q_dtype == TTL_DTYPE_F32) {
            launch_store<HD, __bf16, float>(ctx, c, b, heads, qkv_dev, tiled, bias_dev, rope_dev, rope_positions, q_dev);
        } else {
            launch_store<HD, __bf16, __bf16>(ctx, c, b, heads, qkv_dev, tiled, bias_dev, rope_dev, rope_positions,
                                             q_dev);
        }
    };
    if (cache->head_dim == 64) {
        launch(std::integral_constant<int, 64>());
    } else {
        launch(std::integral_constant<int, 128>());
    }
    TTL_LAUNCHED("rope_store_kv4_kernel");
    return TTL_OK;
}

int ttl_kv4_dequantize(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, float *k_dev,
                       float *v_dev) {
    TTL_REQUIRE(ctx, TTL_ERR_INVALID, "ttl_kv4_dequantize: null context");
    const int rc = kv4::check(cache, batch, "ttl_kv4_dequantize");
    if (rc != TTL_OK) {
        return rc;
    }
    TTL_REQUIRE(aligned16(k_dev) && aligned16(v_dev), TTL_ERR_INVALID,
                "ttl_kv4_dequantize: k and v must be 16-byte aligned");
    if (batch->sequences == 0 || batch->tokens == 0 || (!k_dev && !v_dev)) {
        return TTL_OK;
    }
    const uint32_t slices = ttl::blocks_for(size_t(2) * cache->kv_heads * (cache->head_dim / 8), kThreads);
    TTL_REQUIRE(size_t(batch->tokens) * slices <= kMostGroups, TTL_ERR_SHAPE,
                "ttl_kv4_dequantize: %u tokens are too many for one call", batch->tokens);
    TTL_HIP(hipSetDevice(ctx->device));
    const Cache c = kv4::view(cache);
    const Batch b = kv4::view(batch);
    if (cache->head_dim == 64) {
        dequantize_kv4_kernel<64><<<b.tokens * slices, kThreads, 0, ctx->stream>>>(c, b, slices, k_dev, v_dev);
    } else {
        dequantize_kv4_kernel<128><<<b.tokens * slices, kThreads, 0, ctx->stream>>>(c, b, slices, k_dev, v_dev);
    }
    TTL_LAUNCHED("dequantize_kv4_kernel");
    return TTL_OK;
}

}  // extern "C"
