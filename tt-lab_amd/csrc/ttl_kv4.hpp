// The paged 4-bit K/V cache: what its kernels share (the layout is stated with
// ttl_kv4_cache in include/ttlab_hip.h).
#pragma once

#include "ttl_internal.hpp"

namespace kv4 {

constexpr int block = 32;  // values that share an E8M0 byte

struct Cache {
    uint8_t *pool;
    uint32_t kv_heads, pages, page_shift;  // positions per page = 1 << page_shift
    uint32_t record;                       // bytes of one (page, key/value head)
};

struct Batch {
    const int32_t *table, *lengths, *starts;
    uint32_t sequences, tokens, stride, max_length;
};

// Host: checks of the descriptors (a message with `what`), and the forms the kernels take.
int check(const ttl_kv4_cache *cache, const char *what);
int check(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, const char *what);
Cache view(const ttl_kv4_cache *cache);
Batch view(const ttl_kv4_batch *batch);

// An entry of the call's index arrays, which nothing writes while a kernel runs: a scalar load
// where the index is uniform, also in a kernel that stores.
__host__ __device__ inline int32_t entry(const int32_t *p, size_t i) {
#if defined(__HIP_DEVICE_COMPILE__)
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(reinterpret_cast<uintptr_t>(p))[i];
#else
    return p[i];
#endif
}

// What a row of the call's arrays stands for.
enum RowKind : uint32_t {
    kPadding,  // neither read nor written
    kIdle,     // before position 0: zeros
    kBad,      // a sequence too long, or a page outside the pool: NaN
    kToken,
};
struct Row {
    uint32_t kind, sequence, position;
};

// The last sequence whose rows start at or before `row` (starts[0] <= row).
__host__ __device__ inline uint32_t sequence_of(const Batch &b, uint32_t row) {
    uint32_t lo = 0, hi = b.sequences;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (entry(b.starts, mid) <= int32_t(row)) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__host__ __device__ inline Row row_of(const Batch &b, uint32_t row) {
    Row r{kToken, row, 0};
    int32_t end = int32_t(row) + 1;
    if (b.starts) {
        r.sequence = sequence_of(b, row);
        end = entry(b.starts, r.sequence + 1);
        if (entry(b.starts, r.sequence) > int32_t(row) || end <= int32_t(row)) {
            r.kind = kPadding;
            return r;
        }
    }
    const int32_t length = entry(b.lengths, r.sequence);
    const int64_t position = int64_t(length) - (int64_t(end) - int64_t(row));
    if (length <= 0 || position < 0) {
        r.kind = kIdle;
    } else if (uint32_t(length) > b.max_length) {
        r.kind = kBad;
    }
    r.position = uint32_t(position);
    return r;
}

// The page of a position below max_length; false where the table names none of the pool.
__host__ __device__ inline bool page_of(const Cache &c, const Batch &b, uint32_t sequence, uint32_t position,
                                        uint32_t &page) {
    page = uint32_t(entry(b.table, size_t(sequence) * b.stride + (position >> c.page_shift)));
    return page < c.pages;
}

template <int HD>
struct Layout {
    static constexpr uint32_t code_bytes = HD / 2, scale_bytes = HD / block;
    __host__ __device__ static constexpr uint32_t record(uint32_t page_shift) {
        return (2 * code_bytes + 2 * scale_bytes) << page_shift;
    }
    // offsets in a record
    __device__ static uint32_t k_codes(uint32_t slot) { return slot * code_bytes; }
    __device__ static uint32_t v_codes(uint32_t page_shift, uint32_t slot) {
        return (code_bytes << page_shift) + slot * code_bytes;
    }
    __device__ static uint32_t k_scales(uint32_t page_shift, uint32_t slot) {
        return ((2 * code_bytes) << page_shift) + slot * scale_bytes;
    }
    __device__ static uint32_t v_scales(uint32_t page_shift, uint32_t slot) {
        return ((2 * code_bytes + scale_bytes) << page_shift) + slot * scale_bytes;
    }
};

__device__ inline uint8_t *record_of(const Cache &c, uint32_t page, uint32_t kv_head) {
    return c.pool + (size_t(page) * c.kv_heads + kv_head) * c.record;
}

// An E8M0 byte as the scale operand of the conversions: 2^(byte - 127); byte 255 is an
// infinity there and converts every code to NaN.
__device__ inline float scale_of(uint32_t byte) {
    return __uint_as_float(byte << 23);
}

// The 8 values of a dword of codes.
__device__ inline void values8(uint32_t word, float scale, float (&v)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
    v[0] = a[0];
    v[1] = a[1];
    v[2] = b[0];
    v[3] = b[1];
    v[4] = c[0];
    v[5] = c[1];
    v[6] = d[0];
    v[7] = d[1];
}

}  // namespace kv4
