// Attention over the paged 4-bit K/V cache: one token per sequence, and runs of tokens.
//
// A key/value head's queries are its group's heads of the sequence's new tokens, flattened
// (token, head) and taken in blocks.  Per chunk of 64 positions and tile of 16 queries:
//  - S^T (positions x queries) = K Q^T on v_mfma_f32_16x16x32_bf16, then the online softmax of
//    each query (a column of S^T) in units of log 2;
//  - O^T (dims x queries) += V^T P^T on v_mfma_f32_16x16x32_f16.
// Lane (n, g) = (l % 16, l / 16) of a wave holds 8 values of A row n and B column n for 8 of the
// instruction's 32 K indices, the same for both, and receives D rows 4g..4g+3 of column n.
//
// K: lane group g takes a quarter of the head's dims, g HD/4 .. of position n of a tile, which
// lie next to each other in the cache and in one block, so the codes go from memory to bf16 in
// the lane that multiplies them, the scale folded in (exact: E2M1 x 2^e is a bf16).
// V: its K index is the position, and neighbouring codes of a lane's operand would have
// different scales, so V is converted in the layout it is stored in (dims side by side) to f16
// in LDS, and read back transposed (ds_read_b64_tr_b16: 16 lanes take a 4 x 16 block, lane n its
// column n).  The lane's 8 positions are those of its own rows of two S^T tiles, so the
// weights never leave their registers.
//
// Numerics: K and bf16 queries are exact in bf16, f32 queries three bf16 planes (24 bits).  The
// weights, at most 1 and held times 2^15, are rounded to f16 for a bf16 output (2^-11, an eighth
// of the output's own rounding) and to two f16 planes for an f32 one (2^-22; weights below
// 2^-29 of the largest lose more of themselves, 2^-40 of the largest).  V is exact in f16 where
// its scale bytes are 104..140 (subnormals included: the matrix cores keep them); a chunk with
// another one takes V as bf16, exact for every byte, and three bf16 planes of the weights.
// Maxima, sums and outputs are f32.
#include "ttl_kv4.hpp"
#include "ttl_mfma.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using kv4::Batch;
using kv4::Cache;
using kv4::Layout;
using mf::bf16x8;
using mf::f16x8;
using mf::f32x4;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kChunk = 64, kTiles = kChunk / 16;
constexpr uint32_t kWaves = 4, kThreads = kWaves * 64;
constexpr float kLog2e = 0x1.715476p+0f, kLog2eLo = 0x1.4ae0cp-26f;  // log2 e = their sum
constexpr uint32_t kF16First = 104, kF16Last = 140;                  // scale bytes of V on the f16 path
constexpr float kWeightShift = 15.0f;                               // weights are held times 2^15

struct Params {
    const float *sinks;
    uint32_t heads, group, window;
    float c;      // |scale| log2 e
    float c_lo;   // (|scale| log2 e - c) / c
    bool negate;  // the scale is negative: the queries change their sign instead
};

// How a call is cut: blocks of `queries` queries of a sequence and key/value head, each
// block's chunks in runs of `run` chunks, `splits` at most.
struct Plan {
    uint32_t queries, blocks, run, splits;
    float *o;      // [split][row][head][HD], where a block has more than one run
    float2 *bl;    // [split][row][head]: offset, sum
};

// ---- which queries and positions a block has -----------------------------------------------

struct Block {
    uint32_t sequence, row0, rows;     // the sequence's rows
    uint32_t query0;                   // the block's first query of the sequence
    int32_t position0;                 // of the sequence's first row (negative: idle rows)
    uint32_t first_chunk, chunks;      // none: no row of the block sees a position
    uint32_t lo, hi;                   // the positions that its rows see
    bool exists, bad;
};

__device__ inline Block block_span(const Batch &b, const Params &a, uint32_t queries, Block k) {
    const int32_t length = b.lengths[k.sequence];
    k.position0 = length - int32_t(k.rows);
    k.bad = length > 0 && uint32_t(length) > b.max_length;
    const uint32_t last = min(k.query0 + queries, k.rows * a.group) - 1;
    const int32_t p0 = max(k.position0 + int32_t(k.query0 / a.group), 0), p1 = k.position0 + int32_t(last / a.group);
    k.chunks = 0;
    if (length > 0 && p1 >= 0 && !k.bad) {
        k.hi = uint32_t(p1);
        k.lo = a.window && uint32_t(p0) + 1 > a.window ? uint32_t(p0) + 1 - a.window : 0;
        k.first_chunk = k.lo / kChunk;
        k.chunks = k.hi / kChunk - k.first_chunk + 1;
    }
    return k;
}

// Block `index` of a key/value head.  Sequence s of a ragged batch has its blocks from index
// starts[s] group / queries + s on: rounded down, the sequences' blocks never overlap, and no
// running sum of their numbers is needed (at most one index per sequence stays unused).
__device__ inline Block block_of(const Batch &b, const Params &a, uint32_t queries, uint32_t index) {
    Block k{};
    uint32_t within;
    if (!b.starts) {
        const uint32_t per = (a.group + queries - 1) / queries;
        k.sequence = index / per;
        within = index % per;
        k.row0 = k.sequence;
        k.rows = 1;
    } else {
        uint32_t lo = 0, hi = b.sequences;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const uint32_t s = uint32_t(max(b.starts[mid], 0));
            if (uint64_t(s) * a.group / queries + mid <= index) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        k.sequence = lo;
        k.row0 = min(uint32_t(max(b.starts[lo], 0)), b.tokens);
        const uint32_t end = min(uint32_t(max(b.starts[lo + 1], 0)), b.tokens);
        k.rows = end > k.row0 ? end - k.row0 : 0;
        const uint64_t base = uint64_t(k.row0) * a.group / queries + lo;
        if (index < base) {
            return k;
        }
        within = uint32_t(index - base);
    }
    if (uint64_t(within) * queries >= uint64_t(k.rows) * a.group) {
        return k;
    }
    k.exists = true;
    k.query0 = within * queries;
    return block_span(b, a, queries, k);
}

// ---- the cache's codes as MFMA operands ------------------------------------------------------

// What a lane takes of a chunk: of each 16-position tile, position n, a quarter of the head.
template <int HD>
struct Codes {
    static constexpr int words = HD / 32;  // dwords of 8 codes
    uint32_t w[kTiles][words];
    uint32_t scale[kTiles];
};

template <int HD>
__device__ __attribute__((always_inline)) inline void load_words(const uint8_t *p, uint32_t (&w)[HD / 32]) {
    if constexpr (HD == 64) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x;
        w[1] = x.y;
    } else {
        const uint4 x = *reinterpret_cast<const uint4 *>(p);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    }
}

// Where a chunk's tiles lie: the record of each tile's page and its first slot there.  Tiles
// without a position of lo..hi take the nearest that has.  Pages of 64 positions and more hold
// a chunk whole (TP = 1 look-up); smaller ones TP = 4 tiles apart.
template <int TP>
struct Places {
    uint32_t page[TP];
};
template <int TP>
__device__ __attribute__((always_inline)) inline Places<TP> places_of(const Cache &c, const int32_t *table,
                                                                      uint32_t chunk, uint32_t lo, uint32_t hi) {
    Places<TP> p;
#pragma unroll
    for (uint32_t i = 0; i < TP; ++i) {
        const uint32_t tile = TP == 1 ? chunk * kTiles : min(max(chunk * kTiles + i, lo / 16), hi / 16);
        p.page[i] = uint32_t(table[tile >> (c.page_shift - 4)]);
    }
    return p;
}

// A lane's offsets in a record's tile.
template <int HD>
struct LaneOffsets {
    uint32_t code, scale;
    __device__ LaneOffsets(uint32_t n, uint32_t g)
        : code(n * Layout<HD>::code_bytes + g * (HD / 8)), scale(n * Layout<HD>::scale_bytes + g * (HD / 4) / 32) {}
};

template <int HD, int TP>
__device__ __attribute__((always_inline)) inline void load_chunk(const Cache &c, uint32_t kv_head,
                                                                 const Places<TP> &places, uint32_t chunk, uint32_t lo,
                                                                 uint32_t hi, const LaneOffsets<HD> &at, Codes<HD> &k,
                                                                 Codes<HD> &v) {
    using L = Layout<HD>;
    const uint32_t mask = (1u << c.page_shift) - 1;
    const uint8_t *kp = nullptr, *vp = nullptr, *ks = nullptr, *vs = nullptr;  // uniform
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
        if (TP != 1 || i == 0) {
            const uint32_t tile = TP == 1 ? chunk * kTiles : min(max(chunk * kTiles + i, lo / 16), hi / 16);
            const uint32_t page = places.page[i], slot = (tile * 16) & mask;
            const uint8_t *rec = kv4::record_of(c, page < c.pages ? page : 0u, kv_head);
            kp = rec + L::k_codes(slot);
            vp = rec + L::v_codes(c.page_shift, slot);
            ks = rec + L::k_scales(c.page_shift, slot);
            vs = rec + L::v_scales(c.page_shift, slot);
        }
        const uint32_t tile_code = TP == 1 ? i * 16 * L::code_bytes : 0, tile_scale = TP == 1 ? i * 16 * L::scale_bytes : 0;
        load_words<HD>(kp + (at.code + tile_code), k.w[i]);
        load_words<HD>(vp + (at.code + tile_code), v.w[i]);
        k.scale[i] = ks[at.scale + tile_scale];
        v.scale[i] = vs[at.scale + tile_scale];
    }
}

// What load_chunk left to do for chunks at an end of lo..hi or of the pool: keys of a page
// that is not there read as NaN, values outside lo..hi as zeros.
template <int HD, int TP>
__device__ __attribute__((always_inline)) inline void trim_chunk(const Cache &c, const Places<TP> &places,
                                                                 uint32_t chunk, uint32_t lo, uint32_t hi, uint32_t n,
                                                                 Codes<HD> &k, Codes<HD> &v) {
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
        const uint32_t at = chunk * kChunk + 16 * i + n;
        const bool in_pool = places.page[TP == 1 ? 0 : i] < c.pages;
        const bool zero = at < lo || at > hi || !in_pool;
        if (!in_pool) {
            k.scale[i] = 255;
        }
        v.scale[i] = zero ? 127u : v.scale[i];
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            v.w[i][s] = zero ? 0u : v.w[i][s];
        }
    }
}

template <int TP>
__device__ __attribute__((always_inline)) inline bool all_in_pool(const Cache &c, const Places<TP> &p) {
    bool in = true;
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        in &= p.page[i] < c.pages;
    }
    return in;
}

// ---- the running softmax of a wave's queries ----------------------------------------------------

template <int HD, int QT>
struct State {
    float b[QT];  // offset: c x the largest score - 15; weights are 2^(c s - b)
    float l[QT];  // the lane's share of their sum
    f32x4 o[QT][HD / 16];  // O^T: dims 16 mt + 4g + i of column n
};

__device__ inline float max_over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float sum_over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ inline uint32_t or_over_groups(uint32_t x) {
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = a[0] | a[1];
    const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return b[0] | b[1];
}

// The lane's query of a tile: the positions it sees (none: last < first).
struct Query {
    int32_t first, last;
};

// Scores to weights: masks, the new maximum, the rescaling of what is there.
template <int HD, int QT>
__device__ __attribute__((always_inline)) inline void softmax_step(f32x4 (&s)[kTiles], State<HD, QT> &st, int qi,
                                                                   const Query &q, bool whole, uint32_t chunk,
                                                                   uint32_t g, float c) {
    if (!whole) {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int32_t at = int32_t(chunk * kChunk + 16 * i + 4 * g) + j;
                s[i][j] = at >= q.first && at <= q.last ? s[i][j] : -INFINITY;
            }
        }
    }
    float m = s[0][0];
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m = fmaxf(m, s[i][j]);
        }
    }
    m = max_over_groups(m);
    // fmaxf drops NaN scores; their weights are NaN all the same
    const float b = fmaxf(st.b[qi], m == -INFINITY ? m : fmaf(m, c, -kWeightShift));
    if (__any(b != st.b[qi])) {
        const float keep = b == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.b[qi] - b);
        st.b[qi] = b;
        st.l[qi] *= keep;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                st.o[qi][mt][j] *= keep;
            }
        }
    }
    const float base = b == -INFINITY ? 0.0f : b;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i][j], c, -base));
            s[i][j] = p;
            sum += p;
        }
    }
    st.l[qi] += sum;
}

template <class V>
struct Planes;
template <>
struct Planes<f16x8> {
    typedef _Float16 type2 __attribute__((ext_vector_type(2)));
};
template <>
struct Planes<bf16x8> {
    typedef __bf16 type2 __attribute__((ext_vector_type(2)));
};

// 8 f32 values as P planes, each the remainder rounded.
template <class V, int P>
__device__ __attribute__((always_inline)) inline void split(const float (&x)[8], V (&out)[P]) {
    using T2 = typename Planes<V>::type2;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a = x[e], b = x[e + 1];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const T2 w = __builtin_convertvector(f32x2{a, b}, T2);
            out[p][e] = w[0];
            out[p][e + 1] = w[1];
            if (p + 1 < P) {
                a -= float(w[0]);
                b -= float(w[1]);
            }
        }
    }
}

// ---- V through LDS --------------------------------------------------------------------------------

// Row stride in 16-bit values: 16 more than the head, so that the four rows of a transposing
// read (and the eight of a 16-byte store) fall into different banks.
template <int HD>
constexpr uint32_t kVStride = HD + 16;

template <int HD, class V>
__device__ __attribute__((always_inline)) inline void stage_values(uint16_t *lds, const Codes<HD> &v, uint32_t n,
                                                                   uint32_t g) {
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
        const float scale = kv4::scale_of(v.scale[i]);
        uint16_t *row = lds + (16 * i + n) * kVStride<HD> + g * (HD / 4);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            *reinterpret_cast<V *>(row + 8 * s) = mf::decode_as<V>(v.w[i][s], scale);
        }
    }
}

// A operand of K step h (positions of tiles 2h and 2h + 1) and dims 16 mt..: the lane's own
// rows 4g..4g+3 of both tiles, of dim 16 mt + n.
template <int HD, class V>
__device__ __attribute__((always_inline)) inline V value_fragment(const uint16_t *lds, int h, int mt, uint32_t n,
                                                                  uint32_t g) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const uint16_t *p = lds + (32 * h + 4 * g + n / 4) * kVStride<HD> + 16 * mt + 4 * (n % 4);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 16 * kVStride<HD>));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(V, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

template <int HD, class V, int PP, int QT>
__device__ __attribute__((always_inline)) inline void weigh_values(const uint16_t *lds, const f32x4 (&s)[QT][kTiles],
                                                                   State<HD, QT> &st, uint32_t n, uint32_t g) {
#pragma unroll
    for (int h = 0; h < int(kTiles) / 2; ++h) {
        V p[QT][PP];
#pragma unroll
        for (int qi = 0; qi < QT; ++qi) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = s[qi][2 * h][j];
                x[4 + j] = s[qi][2 * h + 1][j];
            }
            split<V, PP>(x, p[qi]);
        }
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            const V a = value_fragment<HD, V>(lds, h, mt, n, g);
#pragma unroll
            for (int k = PP - 1; k >= 0; --k) {
#pragma unroll
                for (int qi = 0; qi < QT; ++qi) {
                    st.o[qi][mt] = mf::mfma(a, p[qi][k], st.o[qi][mt]);
                }
            }
        }
    }
}

// ---- queries -------------------------------------------------------------------------------------

__device__ inline void load8(const float *p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x;
    v[1] = a.y;
    v[2] = a.z;
    v[3] = a.w;
    v[4] = b.x;
    v[5] = b.y;
    v[6] = b.z;
    v[7] = b.w;
}
__device__ inline void load8(const __bf16 *p, float (&v)[8]) {
    const bf16x8 x = *reinterpret_cast<const bf16x8 *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = float(x[i]);
    }
}

__device__ inline void store4(float *p, const f32x4 &v) {
    *reinterpret_cast<f32x4 *>(p) = v;
}
__device__ inline void store4(__bf16 *p, const f32x4 &v) {
    *reinterpret_cast<bf16x4 *>(p) = __builtin_convertvector(v, bf16x4);
}

// Planes of a type: of the queries (bf16), of the weights (f16).
template <class T>
constexpr int kQueryPlanes = std::is_same<T, float>::value ? 3 : 1;
template <class T>
constexpr int kWeightPlanes = std::is_same<T, float>::value ? 2 : 1;

// The lane's query as B operand of K step s: dims g HD/4 + 8s .., in K's order.  A value that
// is not finite makes every score NaN.
template <int HD, class T>
__device__ __attribute__((always_inline)) inline void load_query(const T *q, uint32_t g, bool negate,
                                                                 bf16x8 (&out)[HD / 32][kQueryPlanes<T>]) {
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) {
        float v[8];
        load8(q + g * (HD / 4) + 8 * s, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = __builtin_isfinite(v[e]) ? (negate ? -v[e] : v[e]) : __builtin_nanf("");
        }
        split<bf16x8, kQueryPlanes<T>>(v, out[s]);
    }
}

// The output of sums o and l at offset b, with the head's sink in the denominator.
__device__ inline f32x4 with_sink(const Params &a, uint32_t head, float b, f32x4 o, float l) {
    if (a.sinks) {
        const float sink = a.sinks[head];
        // log 2 of the sink's weight, with the bits that f32 rounds off the products
        const float lo = __builtin_fabsf(sink) < 0x1p14f ? sink * kLog2eLo : 0.0f;
        float x = fmaf(sink, kLog2e, -b) + (lo - (b + kWeightShift) * a.c_lo);
        x = x > 0x1p100f ? 0x1p100f : x;
        // a sink far above the scores: the sums move down, as its weight would overflow
        const float down = fmaxf(x - 64.0f, 0.0f), keep = __builtin_amdgcn_exp2f(-down);
        l = fmaf(l, keep, __builtin_amdgcn_exp2f(x - down));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] *= keep;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o[j] /= l;
    }
    return o;
}

// ---- few queries: the waves of a workgroup share them and take the chunks in turn -----------------

template <int HD, int QT, int QP>
struct Wave {
    State<HD, QT> st;
    bf16x8 qf[QT][HD / 32][QP];
    Query mine[QT];
    uint32_t nan_blocks[QT];  // blocks of V (a bit each) that hold a NaN the query sees, by lane
};

// A wave's chunks from `chunk` on, every kWaves-th below `end`.  ODD false: it returns at the
// first chunk with a scale byte of V outside the f16 path's (its number, or one past the
// end); ODD true: it takes every chunk to the end on the bf16 path.  A loop of its own for each
// keeps the running state in registers.
template <int HD, class T, int QT, int TP, bool ODD>
__device__ __attribute__((always_inline)) inline uint32_t walk(const Cache &c, const Params &a, const Block &k,
                                                               const int32_t *table, uint32_t kv_head, uint32_t chunk,
                                                               uint32_t end, Codes<HD> &kc, Codes<HD> &vc,
                                                               Places<TP> here, uint16_t *lds, uint32_t n, uint32_t g,
                                                               Wave<HD, QT, kQueryPlanes<T>> &w) {
    constexpr int NS = HD / 32, QP = kQueryPlanes<T>, PP = kWeightPlanes<T>;
    const LaneOffsets<HD> at(n, g);
    // the smallest last and the largest first position of the block's queries, for whole chunks
    const uint32_t last_min = uint32_t(max(k.position0 + int32_t(k.query0 / a.group), 0));
    const uint32_t first_max = a.window && k.hi + 1 > a.window ? k.hi + 1 - a.window : 0;
    Places<TP> next = places_of<TP>(c, table, min(chunk + kWaves, end - 1), k.lo, k.hi);
    while (true) {
        const uint32_t c0 = chunk * kChunk;
        const bool inside = c0 >= k.lo && c0 + kChunk - 1 <= k.hi;
        const bool whole = c0 >= first_max && c0 + kChunk - 1 <= last_min;
        if (!inside || !all_in_pool(c, here)) {
            trim_chunk<HD, TP>(c, here, chunk, k.lo, k.hi, n, kc, vc);
        }
        if (!ODD) {
            uint32_t far = 0;
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                far = max(far, vc.scale[i] - kF16First);
            }
            if (__any(far > kF16Last - kF16First)) {
                return chunk;
            }
        }
        const uint32_t ahead = min(chunk + kWaves, end - 1);
        Codes<HD> kn, vn;
        load_chunk<HD, TP>(c, kv_head, next, ahead, k.lo, k.hi, at, kn, vn);
        here = next;
        next = places_of<TP>(c, table, min(chunk + 2 * kWaves, end - 1), k.lo, k.hi);

        // S^T
        f32x4 s[QT][kTiles];
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
            const float scale = kv4::scale_of(kc.scale[i]);
#pragma unroll
            for (int ks = 0; ks < NS; ++ks) {
                const bf16x8 kf = mf::decode_step(kc.w[i][ks], scale);
#pragma unroll
                for (int p = QP - 1; p >= 0; --p) {
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi) {
                        s[qi][i] = mf::mfma(kf, w.qf[qi][ks][p],
                                            ks == 0 && p == QP - 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qi][i]);
                    }
                }
            }
        }
        if (ODD) {
            // NaN blocks of a position, a bit each, behind its row (its lanes are n, n + 16,
            // n + 32, n + 48); their values are zeros here
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                const bool nan = vc.scale[i] == 255;
                const uint32_t bits = or_over_groups(nan ? 1u << (g * (HD / 4) / 32) : 0u);
                if (g == 0) {
                    lds[(16 * i + n) * kVStride<HD> + HD] = uint16_t(bits);
                }
                vc.scale[i] = nan ? 127u : vc.scale[i];
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    vc.w[i][x] = nan ? 0u : vc.w[i][x];
                }
            }
            stage_values<HD, bf16x8>(lds, vc, n, g);
        } else {
            stage_values<HD, f16x8>(lds, vc, n, g);
        }
#pragma unroll
        for (int qi = 0; qi < QT; ++qi) {
            softmax_step<HD, QT>(s[qi], w.st, qi, w.mine[qi], whole, chunk, g, a.c);
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        if (ODD) {
            weigh_values<HD, bf16x8, 3, QT>(lds, s, w.st, n, g);
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t bits = lds[(16 * i + 4 * g + j) * kVStride<HD> + HD];
                    const int32_t p = int32_t(c0 + 16 * i + 4 * g) + j;
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi) {
                        w.nan_blocks[qi] |= p >= w.mine[qi].first && p <= w.mine[qi].last ? bits : 0u;
                    }
                }
            }
        } else {
            weigh_values<HD, f16x8, PP, QT>(lds, s, w.st, n, g);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        chunk += kWaves;
        if (chunk >= end) {
            return chunk;
        }
        kc = kn;
        vc = vn;
    }
}

// The walk on the bf16 path, with a copy of the state, so that the other walk's stays in
// registers of its own.
template <int HD, class T, int QT, int TP>
__device__ __attribute__((always_inline)) inline void walk_odd(const Cache &c, const Params &a, const Block &k,
                                                   const int32_t *table, uint32_t kv_head, uint32_t chunk,
                                                   uint32_t end, uint16_t *lds, uint32_t n, uint32_t g,
                                                   Wave<HD, QT, kQueryPlanes<T>> &w) {
    const Places<TP> here = places_of<TP>(c, table, chunk, k.lo, k.hi);
    Codes<HD> kc, vc;
    load_chunk<HD, TP>(c, kv_head, here, chunk, k.lo, k.hi, LaneOffsets<HD>(n, g), kc, vc);
    Wave<HD, QT, kQueryPlanes<T>> mine = w;
    walk<HD, T, QT, TP, true>(c, a, k, table, kv_head, chunk, end, kc, vc, here, lds, n, g, mine);
    w = mine;
}

// What bounds it: at long contexts the cache's bytes.  (Figures with the launch.)
// Waves per SIMD that the kernel's registers leave room for.
template <int HD, class T, int QT>
constexpr int kResident = QT == 2 ? (HD == 64 ? 2 : 1) : HD == 128 ? 2 : std::is_same<T, float>::value ? 3 : 4;

template <int HD, class T, int QT, int TP>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kResident<HD, T, QT>))) void
attention_split_kernel(Cache c, Batch b, Params a, Plan plan, const T *__restrict__ q, T *__restrict__ out) {
    constexpr uint32_t kQueries = 16 * QT, kOStride = HD + 4;
    constexpr uint32_t kVWave = kChunk * kVStride<HD>;  // 16-bit values of one wave
    union Shared {
        uint16_t v[kWaves][kVWave];
        struct {
            float o[kWaves][kQueries][kOStride];
            float b[kWaves][kQueries], l[kWaves][kQueries];
        } join;
    };
    __shared__ __attribute__((aligned(16))) Shared sh;

    const uint32_t run = blockIdx.z, kv_head = blockIdx.y;
    const Block k = block_of(b, a, kQueries, blockIdx.x);
    if (!k.exists) {
        return;
    }
    const uint32_t runs = (k.chunks + plan.run - 1) / plan.run;
    const uint32_t t = threadIdx.x;
    if (run >= runs && !(run == 0 && k.chunks == 0)) {
        return;
    }
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / 64), lane = t % 64, n = lane % 16, g = lane / 16;
    const int32_t *const table = b.table + size_t(k.sequence) * b.stride;
    const uint32_t end = k.first_chunk + min(k.chunks, (run + 1) * plan.run);
    const uint32_t first = k.first_chunk + run * plan.run + wave;

    Wave<HD, QT, kQueryPlanes<T>> w;
    Places<TP> here{};
    Codes<HD> kc, vc;
    if (first < end) {
        here = places_of<TP>(c, table, first, k.lo, k.hi);
        load_chunk<HD, TP>(c, kv_head, here, first, k.lo, k.hi, LaneOffsets<HD>(n, g), kc, vc);
    }
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const uint32_t query = k.query0 + 16 * qi + n, token = k.rows == 1 ? 0u : query / a.group;
        const bool there = query < k.rows * a.group;
        const int32_t position = k.position0 + int32_t(token);
        w.mine[qi].last = there ? position : -1;
        w.mine[qi].first = a.window && position + 1 > int32_t(a.window) ? position + 1 - int32_t(a.window) : 0;
        const uint32_t row = k.row0 + (there ? token : 0u);
        const uint32_t head = kv_head * a.group + (there ? query - token * a.group : 0u);
        load_query<HD, T>(q + (size_t(row) * a.heads + head) * HD, g, a.negate, w.qf[qi]);
        w.st.b[qi] = -INFINITY;
        w.st.l[qi] = 0.0f;
        w.nan_blocks[qi] = 0;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            w.st.o[qi][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (first < end) {
        uint16_t *const lds = sh.v[wave];
        const uint32_t at = walk<HD, T, QT, TP, false>(c, a, k, table, kv_head, first, end, kc, vc, here, lds, n, g, w);
        if (at < end) {
            Wave<HD, QT, kQueryPlanes<T>> copy = w;  // (the state itself stays in registers)
            walk_odd<HD, T, QT, TP>(c, a, k, table, kv_head, at, end, lds, n, g, copy);
            w = copy;
        }
    }

    // the waves' states joined through LDS
    __syncthreads();
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const uint32_t poison = or_over_groups(w.nan_blocks[qi]);
        const float l = sum_over_groups(w.st.l[qi]);
        if (g == 0) {
            sh.join.b[wave][16 * qi + n] = w.st.b[qi];
            sh.join.l[wave][16 * qi + n] = l;
        }
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            f32x4 o = w.st.o[qi][mt];
            if (poison >> (mt / 2) & 1) {
                o = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
            *reinterpret_cast<f32x4 *>(&sh.join.o[wave][16 * qi + n][16 * mt + 4 * g]) = o;
        }
    }
    __syncthreads();
    for (uint32_t u = t; u < kQueries * (HD / 4); u += kThreads) {
        const uint32_t local = u / (HD / 4), d = 4 * (u % (HD / 4)), query = k.query0 + local;
        if (query >= k.rows * a.group) {
            break;
        }
        const uint32_t token = query / a.group, row = k.row0 + token, head = kv_head * a.group + query % a.group;
        T *const dst = out + (size_t(row) * a.heads + head) * HD + d;
        if (k.bad || k.position0 + int32_t(token) < 0 || k.chunks == 0) {
            if (run == 0) {
                const float fill = k.bad ? __builtin_nanf("") : 0.0f;
                store4(dst, f32x4{fill, fill, fill, fill});
            }
            continue;
        }
        float top = sh.join.b[0][local];
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) {
            top = fmaxf(top, sh.join.b[w][local]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sh.join.b[w][local] - base);
            const f32x4 x = *reinterpret_cast<const f32x4 *>(&sh.join.o[w][local][d]);
            l = fmaf(sh.join.l[w][local], f, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = fmaf(x[j], f, o[j]);
            }
        }
        if (runs == 1) {
            store4(dst, with_sink(a, head, top, o, l));
        } else {
            const size_t at = (size_t(run) * b.tokens + row) * a.heads + head;
            *reinterpret_cast<f32x4 *>(plan.o + at * HD + d) = o;
            if (d == 0) {
                plan.bl[at] = make_float2(top, l);
            }
        }
    }
}

// ---- the runs of a block joined: a wave per row and head -------------------------------------------

template <int HD, class T>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(Cache c, Batch b, Params a, Plan plan,
                                                                  T *__restrict__ out) {
    constexpr uint32_t kLanes = HD / 4, kParts = 64 / kLanes;  // lanes of an output, runs at a time
    const uint32_t at = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t row = at / a.heads, head = at % a.heads, lane = threadIdx.x % 64;
    if (row >= b.tokens) {
        return;
    }
    const kv4::Row r = kv4::row_of(b, row);
    if (r.kind != kv4::kToken) {
        return;
    }
    Block k{};
    k.sequence = r.sequence;
    k.row0 = b.starts ? uint32_t(max(b.starts[r.sequence], 0)) : r.sequence;
    k.rows = b.starts ? min(uint32_t(max(b.starts[r.sequence + 1], 0)), b.tokens) - k.row0 : 1;
    k.query0 = ((row - k.row0) * a.group + head % a.group) / plan.queries * plan.queries;
    k = block_span(b, a, plan.queries, k);
    const uint32_t runs = (k.chunks + plan.run - 1) / plan.run;
    if (runs <= 1) {
        return;
    }
    const size_t stride = size_t(b.tokens) * a.heads, base = size_t(row) * a.heads + head;
    float top = -INFINITY;
    for (uint32_t i = lane; i < runs; i += 64) {
        top = fmaxf(top, plan.bl[i * stride + base].x);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        top = fmaxf(top, __shfl_xor(top, d));
    }
    const float offset = top == -INFINITY ? 0.0f : top;
    const uint32_t part = lane / kLanes, d = 4 * (lane % kLanes);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
    for (uint32_t i = part; i < runs; i += kParts) {
        const float2 s = plan.bl[i * stride + base];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(plan.o + (i * stride + base) * HD + d);
        const float f = __builtin_amdgcn_exp2f(s.x - offset);
        l = fmaf(s.y, f, l);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = fmaf(x[j], f, o[j]);
        }
    }
#pragma unroll
    for (uint32_t x = kLanes; x < 64; x <<= 1) {
        l += __shfl_xor(l, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] += __shfl_xor(o[j], x);
        }
    }
    if (part == 0) {
        store4(out + base * HD + d, with_sink(a, head, top, o, l));
    }
}

// ---- host -----------------------------------------------------------------------------------------

int check_attention(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, const ttl_kv4_attention *attention,
                    const char *what) {
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

constexpr uint32_t kMaxSplits = 256;

// The cut of a checked call: query tiles per wave by the queries a sequence has on average;
// runs of chunks so that about kTargetGroups workgroups share the longest sequence's walk.
struct Cut {
    uint32_t tiles;
    Plan plan;
    size_t workspace;
};
Cut cut_of(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, const ttl_kv4_attention *attention) {
    constexpr uint64_t kTargetGroups = 2048;
    const uint32_t group = attention->heads / cache->kv_heads;
    Cut cut{};
    const uint64_t queries = uint64_t(batch->tokens) * group;  // of a key/value head
    const uint64_t mean = queries / batch->sequences;
    cut.tiles = mean > 16 ? 2 : 1;
    Plan &p = cut.plan;
    p.queries = 16 * cut.tiles;
    p.blocks = batch->starts ? uint32_t(queries / p.queries + batch->sequences)
                             : batch->sequences * ((group + p.queries - 1) / p.queries);
    uint32_t longest = batch->max_length;
    if (attention->window) {
        // a block's tokens span queries / group + 1 positions at most
        longest = uint32_t(std::min<uint64_t>(longest, uint64_t(attention->window) + p.queries / group + 1));
    }
    const uint32_t chunks = longest / kChunk + (attention->window ? 2 : 1);  // any alignment
    const uint64_t groups = uint64_t(p.blocks) * cache->kv_heads;
    const uint64_t splits =
        std::max<uint64_t>(1, std::min<uint64_t>({kTargetGroups / groups, chunks / kWaves, kMaxSplits}));
    p.run = uint32_t((chunks + splits - 1) / splits);
    p.run = (p.run + kWaves - 1) / kWaves * kWaves;
    p.splits = (chunks + p.run - 1) / p.run;
    if (p.splits > 1) {
        const size_t rows = size_t(p.splits) * batch->tokens * attention->heads;
        cut.workspace = rows * (cache->head_dim * sizeof(float) + sizeof(float2));
    }
    return cut;
}

int run_attention(ttl_ctx *ctx, const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                  const ttl_kv4_attention *attention, const void *q, void *out, void *workspace,
                  size_t workspace_bytes, const char *what) {
    TTL_REQUIRE(ctx, TTL_ERR_INVALID, "%s: null context", what);
    const int rc = check_attention(cache, batch, attention, what);
    if (rc != TTL_OK) {
        return rc;
    }
    if (batch->sequences == 0 || batch->tokens == 0) {
        return TTL_OK;
    }
    TTL_REQUIRE(q && out, TTL_ERR_INVALID, "%s: null argument", what);
    TTL_REQUIRE(((uintptr_t(q) | uintptr_t(out)) & 15) == 0, TTL_ERR_INVALID, "%s: q and out must be 16-byte aligned",
                what);
    Cut cut = cut_of(cache, batch, attention);
    TTL_REQUIRE(cut.workspace == 0 || (workspace && workspace_bytes >= cut.workspace), TTL_ERR_INVALID,
                "%s: a workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : size_t(0),
                cut.workspace);
    TTL_REQUIRE(cut.workspace == 0 || (uintptr_t(workspace) & 255) == 0, TTL_ERR_INVALID,
                "%s: the workspace must be 256-byte aligned", what);
    const uint64_t groups = uint64_t(cut.plan.blocks) * cache->kv_heads * cut.plan.splits;
    TTL_REQUIRE(groups * kThreads <= 0xffffffffu && uint64_t(batch->tokens) * attention->heads <= 0x7fffffffu, TTL_ERR_SHAPE,
                "%s: %u tokens of %u heads are too many for one call", what, batch->tokens, attention->heads);
    TTL_HIP(hipSetDevice(ctx->device));
    const Cache c = kv4::view(cache);
    const Batch b = kv4::view(batch);
    const double scale = std::fabs(double(attention->scale)) * 1.4426950408889634;
    Params a{};
    a.sinks = attention->sinks;
    a.heads = attention->heads;
    a.group = attention->heads / cache->kv_heads;
    a.window = std::min(attention->window, 1u << 30);
    // (a scale of zero still has to leave masked scores, -infinity, what they are)
    a.c = std::max(float(scale), 0x1p-140f);
    a.c_lo = scale > 0x1p-120 ? float((scale - double(a.c)) / double(a.c)) : 0.0f;
    a.negate = attention->scale < 0.0f;
    Plan p = cut.plan;
    if (p.splits > 1) {
        p.o = static_cast<float *>(workspace);
        p.bl = reinterpret_cast<float2 *>(p.o + size_t(p.splits) * b.tokens * a.heads * cache->head_dim);
    }
    const auto launch = [&](auto hd, auto zero) {
        constexpr int HD = decltype(hd)::value;
        using T = decltype(zero);
        const T *qt = static_cast<const T *>(q);
        T *ot = static_cast<T *>(out);
        const dim3 grid(p.blocks, c.kv_heads, p.splits);
        const bool big = c.page_shift >= 6;
        const auto split = [&](auto tiles) {
            constexpr int QT = decltype(tiles)::value;
            if (big) {
                attention_split_kernel<HD, T, QT, 1><<<grid, kThreads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            } else {
                attention_split_kernel<HD, T, QT, 4><<<grid, kThreads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            }
        };
        if (cut.tiles == 1) {
            split(std::integral_constant<int, 1>());
        } else {
            split(std::integral_constant<int, 2>());
        }
        if (p.splits > 1) {
            attention_join_kernel<HD, T><<<ttl::blocks_for(size_t(b.tokens) * a.heads, kWaves), kThreads, 0,
                                           ctx->stream>>>(c, b, a, p, ot);
        }
    };
    if (cache->head_dim == 64) {
        attention->dtype == TTL_DTYPE_F32 ? launch(std::integral_constant<int, 64>(), float())
                                          : launch(std::integral_constant<int, 64>(), __bf16());
    } else {
        attention->dtype == TTL_DTYPE_F32 ? launch(std::integral_constant<int, 128>(), float())
                                          : launch(std::integral_constant<int, 128>(), __bf16());
    }
    TTL_LAUNCHED(what);
    return TTL_OK;
}

}  // namespace

extern "C" {

size_t ttl_attention_kv4_workspace_bytes(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch,
                                         const ttl_kv4_attention *attention) {
    if (check_attention(cache, batch, attention, "ttl_attention_kv4_workspace_bytes") != TTL_OK ||
        batch->sequences == 0 || batch->tokens == 0) {
        return 0;
    }
    return cut_of(cache, batch, attention).workspace;
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
