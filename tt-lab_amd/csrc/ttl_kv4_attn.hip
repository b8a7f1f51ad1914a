// Attention over the paged 4-bit K/V cache: one token per sequence, and runs of tokens.
//
// A key/value head's queries are its group's heads of the sequence's new tokens, flattened
// (token, head) and taken in blocks.  Per chunk of 64 positions and tile of 16 queries:
//  - S^T (positions x queries) = K Q^T on v_mfma_f32_16x16x32_bf16, then the online softmax of
//    each query (a column of S^T) in units of log 2;
//  - O^T (dims x queries) += V^T P^T on the same instruction.
// Lane (n, g) = (l % 16, l / 16) of a wave holds 8 values of A row n and B column n for 8 of the
// instruction's 32 K indices, the same for both, and receives D rows 4g..4g+3 of column n.
//
// K: lane group g takes a quarter of the head's dims, g HD/4 .. of position n of a tile, which
// lie next to each other in the cache and in one block, so the codes go from memory to bf16 in
// the lane that multiplies them, the scale folded in (exact: E2M1 x 2^e is a bf16).
// V: its K index is the position, and neighbouring codes of a lane's operand would have
// different scales, so V is converted in the layout it is stored in (dims side by side) to bf16
// in LDS, and read back transposed (ds_read_b64_tr_b16: 16 lanes take a 4 x 16 block, lane n its
// column n).  The lane's 8 positions are those of its own rows of two S^T tiles, so the
// weights never leave their registers.
//
// Numerics: K, V and bf16 queries are exact in bf16, f32 queries three bf16 planes (24 bits).  The
// weights go into the product with V as bf16 planes, which keep f32's range: three for an f32
// output (2^-24 of a weight), two for a bf16 one (2^-16, where the output's own rounding is 2^-8).
// Maxima, sums and outputs are f32.  A NaN block of V would reach rows that do not see it (a weight
// of zero times NaN), so its values are zeros in LDS and the queries that see it are noted apart.
//
// What bounds them (a large copy moves 5.1 TB/s here, a large bf16 product 1.23 PFLOP/s).  One
// token a sequence: the codes are read once; 128 sequences at 4096 (289 MB, f32 queries) take 77
// us with their join, 3.8 TB/s, 64 ragged ones up to 8192 (151 MB, bf16) 49 us, 3.1 TB/s: the vector
// instructions of conversion and softmax, 29% (bf16) and 42% (f32) of the cycles, against loads
// that 2 or 3 waves a SIMD keep in flight.  Prompts: the vector instructions, 57% of the cycles (an
// exponential a score costs as much as three multiply-adds, its split into two planes as two and a
// half), next to the products' 26%: 4096 tokens of 64 bf16 heads of 64 take 313 us, 440 TFLOP/s
// (251 with the weights as one f16 plane, which lost those 2^-32 and less of the largest).
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
using mf::f32x4;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kChunk = 64, kTiles = kChunk / 16;
constexpr uint32_t kWaves = 4, kThreads = kWaves * 64;
constexpr float kLog2e = 0x1.715476p+0f, kLog2eLo = 0x1.4ae0cp-26f;  // log2 e = their sum
// A weight is held as 2^-8 when it is the largest seen, and grows to 1 at most: what sums up in f32
// is never more than the values' own sum, and few large values have room.
constexpr float kWeightShift = -8.0f;

// How a wave's 16 columns are used (M): kHalf for 8 queries or fewer, columns 8..15 the same
// queries on the other half of the chunk (so that no lane weighs scores that nobody asked for:
// 128 f32 sequences at 4096 in 80 instead of 85 us, level in bf16);
// kOne and kTwo for 16 queries, and 32 in two column tiles.
constexpr int kHalf = 0, kOne = 1, kTwo = 2;
template <int M>
struct Mode {
    static constexpr int columns = M == kHalf ? 1 : M;            // column tiles
    static constexpr int halves = M == kHalf ? 2 : 1;
    static constexpr int tiles = 4 / halves;                      // position tiles of a lane's column
    static constexpr uint32_t queries = M == kHalf ? 8 : 16 * columns;
};

struct Params {
    const float *sinks;
    uint32_t heads, group, window;
    float c;      // |scale| log2 e
    float c_lo;   // (|scale| log2 e - c) / c
    bool negate;  // the scale is negative: the queries change their sign instead
};

// How a call is cut.  A block is up to `queries` queries of a sequence and key/value head; its
// chunks count in units of `unit`.  The units of all blocks in a row are
// divided evenly among `shares` workgroups per key/value head, whatever the lengths are: a share
// takes the end of one block, whole ones, and the beginning of another.  A block that one
// share has whole is written by it; of the others every share leaves its part in `o` and `bl`
// (place 1 where it holds the block's beginning, 0 elsewhere) for the join.
struct Plan {
    uint32_t queries, blocks, shares, unit;
    bool single;   // a share is a block, nothing is joined
    float *o;      // [kv head][share][2][queries][HD]
    float2 *bl;    // [kv head][share][2][queries]: offset, sum
    uint2 *span;   // [block]: its first and last share
};

// ---- which queries and positions a block has -----------------------------------------------

struct Block {
    uint32_t sequence, row0, rows;     // the sequence's rows, those behind the arrays' end left out
    uint32_t query0;                   // the block's first query of the sequence
    int32_t position0;                 // of the sequence's first row (negative: idle rows)
    uint32_t first_chunk, chunks;      // none: no row of the block sees a position
    uint32_t lo, hi;                   // the positions that its rows see
    bool exists, bad;
};

// `all` rows: with those left out, which have the last positions.
__device__ inline Block block_span(const Batch &b, const Params &a, uint32_t queries, Block k, uint32_t all) {
    const int32_t length = max(kv4::entry(b.lengths, k.sequence), 0);
    k.position0 = length - int32_t(all);
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

__device__ inline uint32_t units_of(const Plan &plan, const Block &k) {
    return plan.unit == 1 ? k.chunks : (k.chunks + kWaves - 1) / kWaves;
}

// Block `index` of a key/value head.  Sequence s of a ragged batch has its blocks from index
// starts[s] group / queries + s on: rounded down, the sequences' blocks never overlap, and no
// running sum of their numbers is needed (at most one index per sequence stays unused).
__device__ inline Block block_of(const Batch &b, const Params &a, uint32_t queries, uint32_t index) {
    Block k{};
    uint32_t within, all = 1;
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
            const uint32_t s = uint32_t(max(kv4::entry(b.starts, mid), 0));
            if (uint64_t(s) * a.group / queries + mid <= index) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        k.sequence = lo;
        k.row0 = min(uint32_t(max(kv4::entry(b.starts, lo), 0)), b.tokens);
        const uint32_t end = uint32_t(max(kv4::entry(b.starts, lo + 1), 0));
        all = end > k.row0 ? end - k.row0 : 0;
        k.rows = min(all, b.tokens - k.row0);
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
    return block_span(b, a, queries, k, all);
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
        p.page[i] = uint32_t(kv4::entry(table, tile >> (c.page_shift - 4)));
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

// The codes and scales of a chunk's K or V.
template <int HD, int TP, bool V>
__device__ __attribute__((always_inline)) inline void load_codes(const Cache &c, const uint8_t *head, size_t page_bytes,
                                                                 const Places<TP> &places, uint32_t chunk, uint32_t lo,
                                                                 uint32_t hi, const LaneOffsets<HD> &at, Codes<HD> &x) {
    using L = Layout<HD>;
    const uint32_t mask = (1u << c.page_shift) - 1;
    const uint8_t *codes = nullptr, *scales = nullptr;  // uniform
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
        if (TP != 1 || i == 0) {
            const uint32_t tile = TP == 1 ? chunk * kTiles : min(max(chunk * kTiles + i, lo / 16), hi / 16);
            const uint32_t page = places.page[i], slot = (tile * 16) & mask;
            const uint8_t *rec = head + (page < c.pages ? page : 0u) * page_bytes;
            codes = rec + (V ? L::v_codes(c.page_shift, slot) : L::k_codes(slot));
            scales = rec + (V ? L::v_scales(c.page_shift, slot) : L::k_scales(c.page_shift, slot));
        }
        const uint32_t tile_code = TP == 1 ? i * 16 * L::code_bytes : 0;
        const uint32_t tile_scale = TP == 1 ? i * 16 * L::scale_bytes : 0;
        load_words<HD>(codes + (at.code + tile_code), x.w[i]);
        x.scale[i] = scales[at.scale + tile_scale];
    }
}

// What load_codes left to do for chunks at an end of lo..hi or of the pool: keys of a page
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

template <int HD, int M>
struct State {
    float b[Mode<M>::columns];  // offset: c x a large score + 8; weights are 2^(c s - b), 1 at most
    float l[Mode<M>::columns];  // the lane's share of their sum
    f32x4 o[Mode<M>::columns][HD / 16];  // O^T: dims 16 mt + 4g + i of column n
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

// Scores to weights, in place.  The offset follows the largest score lazily: it is set anew (and
// what is there rescaled) only when a weight would pass 1, or before any score was seen (its
// weights would then be infinite).
// `at`: the position of the lane's first score.
template <int HD, int M>
__device__ __attribute__((always_inline)) inline void softmax_step(f32x4 (&s)[Mode<M>::columns][Mode<M>::tiles],
                                                                   State<HD, M> &st,
                                                                   const Query (&q)[Mode<M>::columns], bool whole,
                                                                   int32_t at, float c) {
    constexpr int NT = Mode<M>::tiles, QT = Mode<M>::columns;
    if (!whole) {
        asm volatile("" : "+v"(at));  // (the positions are computed here, not for every chunk)
#pragma unroll
        for (int qi = 0; qi < QT; ++qi) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int32_t p = at + 16 * i + j;
                    s[qi][i][j] = p >= q[qi].first && p <= q[qi].last ? s[qi][i][j] : -INFINITY;
                }
            }
        }
    }
    float m[QT];
    bool far = false;
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        m[qi] = s[qi][0][0];  // (fmaxf drops NaN scores; their weights are NaN all the same)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m[qi] = fmaxf(m[qi], s[qi][i][j]);
            }
        }
        far |= fmaf(m[qi], c, -st.b[qi]) > 0.0f;
    }
    if (__any(far)) {
#pragma unroll
        for (int qi = 0; qi < QT; ++qi) {
            const float x = max_over_groups(m[qi]);
            const float b = fmaxf(st.b[qi], x == -INFINITY ? x : fmaf(x, c, -kWeightShift));
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
    }
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const float base = st.b[qi] == -INFINITY ? 0.0f : st.b[qi];
        f32x4 x;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[qi][i][j] = __builtin_amdgcn_exp2f(fmaf(s[qi][i][j], c, -base));
                x[j] = i ? x[j] + s[qi][i][j] : s[qi][i][j];
            }
        }
        st.l[qi] += (x[0] + x[1]) + (x[2] + x[3]);
    }
}

// 8 f32 values as P bf16 planes, each the remainder rounded.
template <int P>
__device__ __attribute__((always_inline)) inline void split(const float (&x)[8], bf16x8 (&out)[P]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a = x[e], b = x[e + 1];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const mf::bf16x2 w = __builtin_convertvector(f32x2{a, b}, mf::bf16x2);
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

// Rows of HD 16-bit values, a row's 16-byte pieces in an order of their own, in which 16 rows of
// a piece (16-byte stores and reads) and 8 rows of two neighbouring pieces (transposing reads)
// lie in 64 different banks.  Where piece c of `row` begins, in values:
template <int HD>
__device__ __attribute__((always_inline)) inline uint32_t piece_at(uint32_t row, uint32_t c) {
    const uint32_t turn = HD == 64 ? (row / 2) % 4 : row % 8;
    return row * HD + (((c / 2) ^ turn) * 2 + ((c % 2) ^ (row / 8 % 2))) * 8;
}

template <int HD>
__device__ __attribute__((always_inline)) inline void stage_values(uint16_t *lds, const Codes<HD> &v, uint32_t n,
                                                                   uint32_t g) {
#pragma unroll
    for (uint32_t i = 0; i < kTiles; ++i) {
        const float scale = kv4::scale_of(v.scale[i]);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            // (rows 16 apart are turned alike)
            *reinterpret_cast<bf16x8 *>(lds + piece_at<HD>(n, g * (HD / 32) + s) + 16 * i * HD) =
                mf::decode_step(v.w[i][s], scale);
        }
    }
}

// A operand of K step h (positions of tiles 2h and 2h + 1) and dims 16 mt..: the lane's own
// rows 4g..4g+3 of both tiles, of dim 16 mt + n.
template <int HD>
__device__ __attribute__((always_inline)) inline bf16x8 value_fragment(const uint16_t *lds, int h, int mt, uint32_t n,
                                                                       uint32_t g) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const uint16_t *p = lds + piece_at<HD>(4 * g + n / 4, 2 * mt + n % 4 / 2) + 4 * (n % 2) + 32 * h * HD;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 16 * HD));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

template <int HD, int PP, int M>
__device__ __attribute__((always_inline)) inline void weigh_values(
    const uint16_t *lds, const f32x4 (&s)[Mode<M>::columns][Mode<M>::tiles], State<HD, M> &st, uint32_t n, uint32_t g) {
    constexpr int QT = Mode<M>::columns;
    // fragments requested together, and a batch ahead beside the three planes of f32 queries' weights
    // (512 tokens at 2048: 69.4 against 70.4 us); beside two it is level to slower
    constexpr int kSteps = int(kTiles) / 2, kBatch = 4, kBuffers = PP == 3 ? 2 : 1;
    constexpr int kFragments = kSteps * (HD / 16);
    const auto fragment = [&](int f) __attribute__((always_inline)) {
        return value_fragment<HD>(lds, f / (HD / 16), f % (HD / 16), n, g);
    };
    bf16x8 a[kBuffers][kBatch];
    const auto request = [&](int f0) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < kBatch; ++f) {
            a[f0 / kBatch % kBuffers][f] = fragment(f0 + f);
        }
    };
    if (kBuffers == 2) {
        request(0);
    }
    bf16x8 p[QT][PP];
#pragma unroll
    for (int f0 = 0; f0 < kFragments; f0 += kBatch) {
        const int h = f0 / (HD / 16);
        if (f0 % (HD / 16) == 0) {
#pragma unroll
            for (int qi = 0; qi < QT; ++qi) {
                constexpr int kOwn = M == kHalf ? 0 : 2;
                float x[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[j] = s[qi][kOwn * h][j];
                    x[4 + j] = s[qi][kOwn * h + 1][j];
                }
                split(x, p[qi]);
                if (M == kHalf) {  // the lane's tiles are K step 0 in columns 0..7, step 1 in 8..15
#pragma unroll
                    for (int k = 0; k < PP; ++k) {
                        const mf::u32x4 w = __builtin_bit_cast(mf::u32x4, p[qi][k]);
                        p[qi][k] = __builtin_bit_cast(bf16x8, int(n / 8) == h ? w : mf::u32x4{0u, 0u, 0u, 0u});
                    }
                }
            }
        }
        const int ahead = f0 + (kBuffers - 1) * kBatch;
        if (ahead < kFragments) {
            request(ahead);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = PP - 1; k >= 0; --k) {
#pragma unroll
            for (int f = 0; f < kBatch; ++f) {
                const int mt = (f0 + f) % (HD / 16);
#pragma unroll
                for (int qi = 0; qi < QT; ++qi) {
                    st.o[qi][mt] = mf::mfma(a[f0 / kBatch % kBuffers][f], p[qi][k], st.o[qi][mt]);
                }
            }
        }
    }
}

// ---- queries -------------------------------------------------------------------------------------

__device__ inline void store4(float *p, const f32x4 &v) {
    *reinterpret_cast<f32x4 *>(p) = v;
}
__device__ inline void store4(__bf16 *p, const f32x4 &v) {
    *reinterpret_cast<bf16x4 *>(p) = __builtin_convertvector(v, bf16x4);
}

// bf16 planes of a type: of the queries, of the weights.
template <class T>
constexpr int kQueryPlanes = std::is_same<T, float>::value ? 3 : 1;
template <class T>
constexpr int kWeightPlanes = std::is_same<T, float>::value ? 3 : 2;

// The lane's query as B operand of K step s: dims g HD/4 + 8s .., in K's order.  A value that
// is not finite makes every score NaN.
template <int HD, class T>
struct RawQuery {
    static constexpr int kLoads = HD / 4 * int(sizeof(T)) / 16;
    mf::u32x4 raw[kLoads];
    __device__ __attribute__((always_inline)) inline void load(const T *q, uint32_t g) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            raw[i] = reinterpret_cast<const mf::u32x4 *>(q + g * (HD / 4))[i];
        }
    }
    __device__ __attribute__((always_inline)) inline float value(int s, int e) const {
        if constexpr (std::is_same<T, float>::value) {
            return __uint_as_float(raw[2 * s + e / 4][e % 4]);
        } else {
            const uint32_t w = raw[s][e / 2];
            return __uint_as_float(e % 2 ? w & 0xffff0000u : w << 16);
        }
    }
    __device__ __attribute__((always_inline)) inline void planes(bool negate,
                                                                 bf16x8 (&out)[HD / 32][kQueryPlanes<T>]) const {
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = value(s, e);
                v[e] = __builtin_isfinite(v[e]) ? (negate ? -v[e] : v[e]) : __builtin_nanf("");
            }
            split(v, out[s]);
        }
    }
};

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

template <int HD, int M, int QP>
struct Wave {
    State<HD, M> st;
    bf16x8 qf[Mode<M>::columns][HD / 32][QP];
    Query mine[Mode<M>::columns];
    uint32_t nan_blocks[Mode<M>::columns];  // blocks of V (a bit each) with a NaN that the query sees, by lane
};

// Where a block's chunks come from.
template <int TP>
struct Source {
    const int32_t *table;
    const uint8_t *head;  // the key/value head's record of page 0
    size_t page_bytes;
    uint32_t lo, hi;
    // the smallest last and the largest first position of the block's queries, for whole chunks
    uint32_t last_min, first_max;
    __device__ Places<TP> places(const Cache &c, uint32_t chunk) const {
        return places_of<TP>(c, table, chunk, lo, hi);
    }
};

// A wave's chunks from `chunk` on, every kWaves-th below `end`; kc and vc hold the first one's
// codes.  The next chunk's K is requested when this one's is multiplied, its V when this one's is
// in LDS, into the same registers.
template <int HD, class T, int M, int TP>
__device__ __attribute__((always_inline)) inline void walk(const Cache &c, const Params &a, const Source<TP> &src,
                                                           uint32_t chunk, uint32_t end, Codes<HD> &kc, Codes<HD> &vc,
                                                           Places<TP> here, Places<TP> next, uint16_t *lds, uint32_t n,
                                                           uint32_t g, Wave<HD, M, kQueryPlanes<T>> &w) {
    constexpr int NS = HD / 32, QP = kQueryPlanes<T>, PP = kWeightPlanes<T>, QT = Mode<M>::columns;
    constexpr int NT = Mode<M>::tiles;
    const LaneOffsets<HD> at(n, g);
    const bool upper = M == kHalf && n >= 8;
    while (true) {
        const uint32_t c0 = chunk * kChunk;
        const bool inside = c0 >= src.lo && c0 + kChunk - 1 <= src.hi;
        const bool whole = c0 >= src.first_max && c0 + kChunk - 1 <= src.last_min;
        if (!inside || !all_in_pool(c, here)) {
            trim_chunk<HD, TP>(c, here, chunk, src.lo, src.hi, n, kc, vc);
        }
        uint32_t largest = vc.scale[0];
#pragma unroll
        for (uint32_t i = 1; i < kTiles; ++i) {
            largest = max(largest, vc.scale[i]);
        }
        const bool nans = __any(largest == 255);
        if (nans) {
            // NaN blocks of a position, a bit each, behind the rows (its lanes are n, n + 16,
            // n + 32, n + 48); their values are zeros from here on
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                const bool nan = vc.scale[i] == 255;
                const uint32_t bits = or_over_groups(nan ? 1u << (g * (HD / 4) / 32) : 0u);
                if (g == 0) {
                    lds[kChunk * HD + 16 * i + n] = uint16_t(bits);
                }
                vc.scale[i] = nan ? 127u : vc.scale[i];
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    vc.w[i][x] = nan ? 0u : vc.w[i][x];
                }
            }
        }
        const uint32_t ahead = min(chunk + kWaves, end - 1);
        here = next;
        next = src.places(c, min(chunk + 2 * kWaves, end - 1));

        // S^T, the tiles side by side: products of one accumulator wait for each other
        f32x4 st[QT][kTiles];
#pragma unroll
        for (int ks = 0; ks < NS; ++ks) {
            bf16x8 kf[kTiles];
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                kf[i] = mf::decode_step(kc.w[i][ks], kv4::scale_of(kc.scale[i]));
            }
#pragma unroll
            for (int p = QP - 1; p >= 0; --p) {
#pragma unroll
                for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi) {
                        st[qi][i] = mf::mfma(kf[i], w.qf[qi][ks][p],
                                             ks == 0 && p == QP - 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : st[qi][i]);
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_codes<HD, TP, false>(c, src.head, src.page_bytes, here, ahead, src.lo, src.hi, at, kc);
        stage_values<HD>(lds, vc, n, g);
        __builtin_amdgcn_sched_barrier(0);
        load_codes<HD, TP, true>(c, src.head, src.page_bytes, here, ahead, src.lo, src.hi, at, vc);

        f32x4 s[QT][NT];
        const int32_t at0 = int32_t(c0 + 4 * g) + (upper ? 32 : 0);
#pragma unroll
        for (int qi = 0; qi < QT; ++qi) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[qi][i][j] = M == kHalf && upper ? st[qi][i + kTiles - NT][j] : st[qi][i][j];
                }
            }
        }
        softmax_step<HD, M>(s, w.st, w.mine, whole, at0, a.c);
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        weigh_values<HD, PP, M>(lds, s, w.st, n, g);
        if (nans) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int32_t p = at0 + 16 * i + j;
                    const uint32_t bits = lds[kChunk * HD + uint32_t(p) - c0];
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi) {
                        w.nan_blocks[qi] |= p >= w.mine[qi].first && p <= w.mine[qi].last ? bits : 0u;
                    }
                }
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        chunk += kWaves;
        if (chunk >= end) {
            return;
        }
    }
}

template <uint32_t W>
struct ShareScan {
    uint32_t sum[W];
    uint32_t block, first;  // the share's first block, and that block's first unit
};

// Workgroups of a CU (waves of a SIMD).  One more would fit with M kHalf, and was slower: 4 instead
// of 3 for bf16 queries 52.8 against 50.9 us (64 ragged sequences up to 8192), 3 instead of 2 for
// f32 83 against 80 us (128 at 4096; 16 bytes of scratch).
template <int HD, class T, int M>
constexpr int kResident = M == kTwo ? (HD == 64 ? 2 : 1) : HD == 128 || std::is_same<T, float>::value ? 2 : 3;

template <int HD, int M>
union Shared {
    static constexpr uint32_t kOStride = HD + 4;
    uint16_t v[kWaves][kChunk * (HD + 1)];  // rows, and a word per row for its NaN blocks
    struct {
        float o[kWaves][16 * Mode<M>::columns][kOStride];
        float b[kWaves][16 * Mode<M>::columns], l[kWaves][16 * Mode<M>::columns];
    } join;
    ShareScan<kWaves> scan;
};

// Units [from, to) of a block: the waves take its chunks in turn, and their states are joined.
// place < 0: the block is whole, its outputs are written; else the place of the share's part.
template <int HD, class T, int M, int TP>
__device__ __attribute__((always_inline)) inline void do_block(const Cache &c, const Batch &b, const Params &a,
                                                               const Plan &plan, const Block &k, uint32_t kv_head,
                                                               uint32_t from, uint32_t to, int place, uint32_t share,
                                                               Shared<HD, M> &sh, const T *q, T *out) {
    constexpr uint32_t kQueries = Mode<M>::queries;
    constexpr int QT = Mode<M>::columns;
    // (opaque: what follows from the lane is computed here again for each block, where the
    // compiler would hold all of it in registers for the whole kernel, and spill)
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / 64), lane = t % 64, n = lane % 16, g = lane / 16;
    Source<TP> src;
    src.table = b.table + size_t(k.sequence) * b.stride;
    src.page_bytes = size_t(c.kv_heads) * c.record;
    src.head = c.pool + size_t(kv_head) * c.record;
    src.lo = k.lo;
    src.hi = k.hi;
    src.last_min = uint32_t(max(k.position0 + int32_t(k.query0 / a.group), 0));
    src.first_max = a.window && k.hi + 1 > a.window ? k.hi + 1 - a.window : 0;
    const uint32_t end = k.first_chunk + min(k.chunks, to * kWaves);
    const uint32_t first = k.first_chunk + from * kWaves + wave;

    Wave<HD, M, kQueryPlanes<T>> w;
    Places<TP> here{}, next{};
    Codes<HD> kc, vc;
    // everything that the first chunk needs is requested before anything is waited for
    if (first < end) {
        here = src.places(c, first);
        next = src.places(c, min(first + kWaves, end - 1));
    }
    RawQuery<HD, T> raw[QT];
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const uint32_t query = k.query0 + (M == kHalf ? n % 8 : 16 * qi + n);
        const uint32_t token = k.rows == 1 ? 0u : query / a.group;
        const bool there = query < k.rows * a.group;
        const int32_t position = k.position0 + int32_t(token);
        w.mine[qi].last = there ? position : -1;
        w.mine[qi].first = a.window && position + 1 > int32_t(a.window) ? position + 1 - int32_t(a.window) : 0;
        const uint32_t row = k.row0 + (there ? token : 0u);
        const uint32_t head = kv_head * a.group + (there ? query - token * a.group : 0u);
        raw[qi].load(q + (size_t(row) * a.heads + head) * HD, g);
        w.st.b[qi] = -INFINITY;
        w.st.l[qi] = 0.0f;
        w.nan_blocks[qi] = 0;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            w.st.o[qi][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (first < end) {
        load_codes<HD, TP, false>(c, src.head, src.page_bytes, here, first, src.lo, src.hi, LaneOffsets<HD>(n, g), kc);
        load_codes<HD, TP, true>(c, src.head, src.page_bytes, here, first, src.lo, src.hi, LaneOffsets<HD>(n, g), vc);
    }
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        raw[qi].planes(a.negate, w.qf[qi]);
    }
    if (first < end) {
        walk<HD, T, M, TP>(c, a, src, first, end, kc, vc, here, next, sh.v[wave], n, g, w);
    }

    // the columns' states joined through LDS
    __syncthreads();
    asm volatile("" : "+v"(t));
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
        float top = -INFINITY;
#pragma unroll
        for (uint32_t x = 0; x < kWaves * Mode<M>::halves; ++x) {
            top = fmaxf(top, sh.join.b[x % kWaves][local + x / kWaves * 8]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < kWaves * Mode<M>::halves; ++x) {
            const uint32_t column = local + x / kWaves * 8;
            const float f = __builtin_amdgcn_exp2f(sh.join.b[x % kWaves][column] - base);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(&sh.join.o[x % kWaves][column][d]);
            l = fmaf(sh.join.l[x % kWaves][column], f, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = fmaf(y[j], f, o[j]);
            }
        }
        if (place < 0) {
            const uint32_t token = k.rows == 1 ? 0u : query / a.group, row = k.row0 + token;
            const uint32_t head = kv_head * a.group + query - token * a.group;
            const bool idle = k.position0 + int32_t(token) < 0;
            store4(out + (size_t(row) * a.heads + head) * HD + d,
                   idle ? f32x4{0.f, 0.f, 0.f, 0.f} : with_sink(a, head, top, o, l));
        } else {
            const size_t at = ((size_t(kv_head) * plan.shares + share) * 2 + uint32_t(place)) * kQueries + local;
            *reinterpret_cast<f32x4 *>(plan.o + at * HD + d) = o;
            if (d == 0) {
                plan.bl[at] = make_float2(top, l);
            }
        }
    }
}

// The outputs of a block whose rows see nothing: zeros, or NaN for a sequence that is too long.
template <int HD, class T>
__device__ inline void fill_block(const Params &a, uint32_t queries, const Block &k, uint32_t kv_head, T *out) {
    for (uint32_t u = threadIdx.x; u < queries * (HD / 4); u += blockDim.x) {
        const uint32_t query = k.query0 + u / (HD / 4), d = 4 * (u % (HD / 4));
        if (query >= k.rows * a.group) {
            break;
        }
        const uint32_t token = query / a.group, row = k.row0 + token, head = kv_head * a.group + query % a.group;
        const float fill = k.bad && k.position0 + int32_t(token) >= 0 ? __builtin_nanf("") : 0.0f;
        store4(out + (size_t(row) * a.heads + head) * HD + d, f32x4{fill, fill, fill, fill});
    }
}

// The part of a share that lies in `block`s, one after the other: `work(k, from, to, place)` does
// units [from, to) of block k.  Called by every thread of a workgroup.
template <int HD, class T, uint32_t W, class Work>
__device__ __attribute__((always_inline)) inline void do_share(const Batch &b, const Params &a, const Plan &plan,
                                                               ShareScan<W> &scan, T *out, const Work &work) {
    const uint32_t share = blockIdx.x, kv_head = blockIdx.y, t = threadIdx.x;
    uint32_t block, unit = 0, from = 0, to, shares = 0;  // the block, its first unit, the share's units
    uint64_t total = 0;
    if (plan.single) {
        block = plan.shares - 1 - share;  // (the blocks with the most positions come last: first of all)
        const Block k = block_of(b, a, plan.queries, block);
        to = units_of(plan, k);
        if (to == 0 && k.exists) {
            fill_block<HD, T>(a, plan.queries, k, kv_head, out);
        }
    } else {
        // every workgroup sums up all blocks' units, and finds where its share begins
        const uint32_t wave = t / 64, lane = t % 64;
        const uint32_t per = (plan.blocks + W * 64 - 1) / (W * 64), mine0 = t * per;
        uint32_t mine = 0;
        for (uint32_t i = mine0; i < min(mine0 + per, plan.blocks); ++i) {
            mine += units_of(plan, block_of(b, a, plan.queries, i));
        }
        uint32_t sum = mine;  // of the lanes up to this one
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t x = __shfl_up(sum, d);
            sum += lane >= d ? x : 0u;
        }
        if (lane == 63) {
            scan.sum[wave] = sum;
        }
        __syncthreads();
        uint32_t before = sum - mine;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const uint32_t x = scan.sum[w];
            before += w < wave ? x : 0u;
            total += x;
        }
        shares = uint32_t(min(uint64_t(plan.shares), total));  // a unit each at least
        if (share >= shares) {
            return;
        }
        from = uint32_t(total * share / shares);
        to = uint32_t(total * (share + 1) / shares);
        if (from >= before && from < before + mine) {
            uint32_t at = before, i = mine0;
            while (true) {
                const uint32_t n = units_of(plan, block_of(b, a, plan.queries, i));
                if (from < at + n) {
                    break;
                }
                at += n;
                ++i;
            }
            scan.block = i;
            scan.first = at;
        }
        __syncthreads();
        block = __builtin_amdgcn_readfirstlane(scan.block);
        unit = __builtin_amdgcn_readfirstlane(scan.first);
        __syncthreads();
    }
    while (unit < to) {
        const Block k = block_of(b, a, plan.queries, block);
        const uint32_t units = units_of(plan, k);
        if (units) {
            const uint32_t x = max(from, unit), y = min(to, unit + units);
            const int place = x == unit && y == unit + units ? -1 : x == unit ? 1 : 0;
            if (place != 0 && !plan.single && kv_head == 0 && t == 0) {
                // the share of a unit u is the last one that begins at u or before
                const uint64_t last = (uint64_t(unit) + units) * shares - 1;
                plan.span[block] = make_uint2(share, uint32_t(last / total));
            }
            work(k, x - unit, y - unit, place);
            __syncthreads();
        }
        unit += units;
        ++block;
    }
}

template <int HD, class T, int M, int TP>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kResident<HD, T, M>))) void
attention_split_kernel(Cache c, Batch b, Params a, Plan plan, const T *__restrict__ q, T *__restrict__ out) {
    __shared__ __attribute__((aligned(16))) Shared<HD, M> sh;
    do_share<HD, T, kWaves>(b, a, plan, sh.scan, out, [&](const Block &k, uint32_t from, uint32_t to, int place) {
        do_block<HD, T, M, TP>(c, b, a, plan, k, blockIdx.y, from, to, place, blockIdx.x, sh, q, out);
    });
}

// ---- many queries: the waves of a workgroup share the chunks, each with queries of its own --------
//
// The waves convert the chunk's tiles of 16 positions to bf16 in LDS, where all of them read them;
// two buffers, so that the next chunk is converted while this one is used, with one barrier a
// chunk.  A tile with a NaN block of V is found when it is converted (a flag a tile, beside the
// buffer).

// Its waves: 8 with one column tile of queries each, four of which convert K and four V; 4 with
// two for f32 queries of 64, whose registers leave room for 8 waves a CU either way (4096
// tokens of 64 heads: 439 against 497 us, though 512 at 2048 69 against 61).  With heads of 128 two
// column tiles spill (2048 tokens of 20 heads: 8 waves 94 against 202 us in f32, 71 against 122 in
// bf16).
template <int HD, class T>
struct Tile {
    static constexpr bool wide = HD == 128 || !std::is_same<T, float>::value;
    static constexpr uint32_t waves = wide ? 8 : 4, threads = waves * 64;
    static constexpr int mode = wide ? kOne : kTwo, parts = wide ? 1 : 2;  // parts: what a wave converts
    static constexpr uint32_t queries = waves * 16 * mode;
    static constexpr int waves_per_simd = wide && HD == 64 ? 4 : 2;
    static constexpr uint32_t groups = waves_per_simd * 4 / waves;  // of a CU
};

template <int HD, class T>
union TileShared {
    struct {
        uint16_t k[2][kChunk * HD], v[2][kChunk * HD];
        uint16_t nan[2][kChunk], nans[2][kTiles];  // NaN blocks of a position, a bit each; tiles that have any
    };
    ShareScan<Tile<HD, T>::waves> scan;
};

// K's or V's codes of one tile of a chunk (position n, a quarter of the head).
template <int HD>
struct TileCodes {
    uint32_t w[HD / 32], scale;
};

// Where the tiles of one part (K or V) and index lie: what is the same in every chunk is added up
// once, the tile's place in its chunk in the lane's offsets (pages of 64 and more hold it at a
// fixed distance), so that a chunk costs few scalar instructions.
template <int HD, int TP>
struct TileSource {
    const uint8_t *codes, *scales;  // uniform: of slot 0 of page 0
    uint32_t code, scale;           // the lane's offsets
    uint32_t page_bytes, mask;      // (kv_heads x record is below 2^24)
    __device__ TileSource(const Cache &c, const Source<TP> &src, const LaneOffsets<HD> &at, uint32_t index, bool v)
        : codes(src.head + (v ? Layout<HD>::v_codes(c.page_shift, 0) : 0)),
          scales(src.head + (v ? Layout<HD>::v_scales(c.page_shift, 0) : Layout<HD>::k_scales(c.page_shift, 0))),
          code(at.code + (TP == 1 ? index * 16 * Layout<HD>::code_bytes : 0)),
          scale(at.scale + (TP == 1 ? index * 16 * Layout<HD>::scale_bytes : 0)),
          page_bytes(c.kv_heads * c.record), mask((1u << c.page_shift) - 1) {}
};

template <int HD, int TP>
__device__ __attribute__((always_inline)) inline void load_tile(const Cache &c, const Source<TP> &src,
                                                                const TileSource<HD, TP> &from, uint32_t chunk,
                                                                uint32_t page, uint32_t index, TileCodes<HD> &x) {
    const uint32_t tile = TP == 1 ? chunk * kTiles : min(max(chunk * kTiles + index, src.lo / 16), src.hi / 16);
    const uint32_t slot = (tile * 16) & from.mask;
    const size_t at = size_t(page < c.pages ? page : 0u) * from.page_bytes;  // uniform
    load_words<HD>(from.codes + (at + slot * Layout<HD>::code_bytes) + from.code, x.w);
    x.scale = (from.scales + (at + slot * Layout<HD>::scale_bytes))[from.scale];
}

// Chunks from `first` on, `count` of them.
struct ChunkRange {
    uint32_t first, count;
    __device__ ChunkRange(uint32_t from, uint32_t end) : first(from), count(end > from ? end - from : 0) {}
    __device__ bool has(uint32_t chunk) const { return chunk - first < count; }
};

// The page of a tile of a chunk.
template <int TP>
__device__ __attribute__((always_inline)) inline uint32_t tile_page(const Cache &c, const Source<TP> &src,
                                                                    uint32_t chunk, uint32_t index) {
    const uint32_t tile = TP == 1 ? chunk * kTiles : min(max(chunk * kTiles + index, src.lo / 16), src.hi / 16);
    return uint32_t(kv4::entry(src.table, tile >> (c.page_shift - 4)));
}

// The lane's quarter of row n.
template <int HD>
__device__ __attribute__((always_inline)) inline void stage_row(uint16_t *rows, uint32_t n, uint32_t g,
                                                                const uint32_t (&w)[HD / 32], uint32_t scale) {
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) {
        *reinterpret_cast<bf16x8 *>(rows + piece_at<HD>(n, g * (HD / 32) + s)) =
            mf::decode_step(w[s], kv4::scale_of(scale));
    }
}

template <int HD, class T, int TP>
__device__ __attribute__((always_inline)) inline void do_tile(const Cache &c, const Batch &b, const Params &a,
                                                              const Plan &plan, const Block &k, uint32_t kv_head,
                                                              uint32_t from, uint32_t to, int place, uint32_t share,
                                                              TileShared<HD, T> &sh, const T *q, T *out) {
    constexpr int M = Tile<HD, T>::mode, KV = Tile<HD, T>::parts;
    constexpr int QT = Mode<M>::columns, NS = HD / 32, QP = kQueryPlanes<T>, PP = kWeightPlanes<T>;
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));  // (as in do_block)
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / 64), lane = t % 64, n = lane % 16, g = lane / 16;
    const uint32_t index = wave % kTiles;  // of the tile that the wave converts
    const auto is_v = [&](int part) __attribute__((always_inline)) { return KV == 2 ? part == 1 : wave >= kTiles; };
    Source<TP> src;
    src.table = b.table + size_t(k.sequence) * b.stride;
    src.page_bytes = size_t(c.kv_heads) * c.record;
    src.head = c.pool + size_t(kv_head) * c.record;
    src.lo = k.lo;
    src.hi = k.hi;
    const LaneOffsets<HD> at(n, g);
    const uint32_t first = k.first_chunk + from, end = k.first_chunk + to;

    // the wave's own queries: which, what they see, and what all and any of them see
    State<HD, M> st;
    bf16x8 qf[QT][NS][QP];
    Query mine[QT];
    uint32_t nan_blocks[QT];
    const uint32_t own = k.query0 + wave * (16 * QT), limit = k.rows * a.group;
    const uint32_t own_last = min(own + 16 * QT, limit) - 1;
    const bool any = own < limit;
    const int32_t p0 = k.position0 + int32_t((any ? own : 0u) / a.group);
    const int32_t p1 = k.position0 + int32_t((any ? own_last : 0u) / a.group);
    // the first position that one at p sees (p may be negative: rows before position 0)
    const auto first_seen = [&](int32_t p) __attribute__((always_inline)) {
        return a.window && p + 1 > int32_t(a.window) ? p + 1 - int32_t(a.window) : 0;
    };
    const uint32_t first_min = uint32_t(first_seen(p0)), first_max = uint32_t(first_seen(p1));
    // the chunks of which some query sees a position, of which all see every one, and that lie
    // in lo..hi whole
    const ChunkRange needed(first_min / kChunk, any && p1 >= 0 ? uint32_t(p1) / kChunk + 1 : 0);
    const ChunkRange whole((first_max + kChunk - 1) / kChunk, p0 >= 0 ? uint32_t(p0 + 1) / kChunk : 0);
    const ChunkRange inside((k.lo + kChunk - 1) / kChunk, (k.hi + 1) / kChunk);
#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const uint32_t query = own + 16 * qi + n, token = query / a.group;
        const bool there = query < limit;
        const int32_t position = k.position0 + int32_t(token);
        mine[qi].last = there ? position : -1;
        mine[qi].first = first_seen(position);
        const uint32_t row = k.row0 + (there ? token : 0u);
        const uint32_t head = kv_head * a.group + (there ? query - token * a.group : 0u);
        RawQuery<HD, T> raw;
        raw.load(q + (size_t(row) * a.heads + head) * HD, g);
        raw.planes(a.negate, qf[qi]);
        st.b[qi] = -INFINITY;
        st.l[qi] = 0.0f;
        nan_blocks[qi] = 0;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            st.o[qi][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    TileCodes<HD> x[KV];
    const TileSource<HD, TP> from_k(c, src, at, index, is_v(0)), from_v(c, src, at, index, is_v(KV - 1));
    const auto load = [&](uint32_t chunk, uint32_t page) __attribute__((always_inline)) {
#pragma unroll
        for (int part = 0; part < KV; ++part) {
            load_tile<HD, TP>(c, src, part ? from_v : from_k, chunk, page, index, x[part]);
        }
    };
    // a page that is not there: keys read as NaN; values outside lo..hi are zeros
    const auto trim = [&](uint32_t chunk, uint32_t page) __attribute__((always_inline)) {
        const uint32_t p = chunk * kChunk + 16 * index + n;
        if (!inside.has(chunk) || page >= c.pages) {
            const bool zero = p < src.lo || p > src.hi || page >= c.pages;
#pragma unroll
            for (int part = 0; part < KV; ++part) {
                if (!is_v(part)) {
                    x[part].scale = page >= c.pages ? 255u : x[part].scale;
                    continue;
                }
                x[part].scale = zero ? 127u : x[part].scale;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    x[part].w[s] = zero ? 0u : x[part].w[s];
                }
            }
        }
    };
    const auto stage = [&](uint32_t buffer, uint32_t chunk, uint32_t page) __attribute__((always_inline)) {
        trim(chunk, page);
        const uint32_t buf = buffer % 2;
#pragma unroll
        for (int part = 0; part < KV; ++part) {
            if (!is_v(part)) {
                stage_row<HD>(sh.k[buf] + 16 * index * HD, n, g, x[part].w, x[part].scale);
                continue;
            }
            const bool nan = x[part].scale == 255, some = __any(nan);
            if (some) {
                const uint32_t bits = or_over_groups(nan ? 1u << (g * (HD / 4) / 32) : 0u);
                x[part].scale = nan ? 127u : x[part].scale;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    x[part].w[s] = nan ? 0u : x[part].w[s];
                }
                if (g == 0) {
                    sh.nan[buf][16 * index + n] = uint16_t(bits);
                }
            }
            if (lane == 0) {
                sh.nans[buf][index] = some ? 1u : 0u;
            }
            stage_row<HD>(sh.v[buf] + 16 * index * HD, n, g, x[part].w, x[part].scale);
        }
    };
    uint32_t page = tile_page<TP>(c, src, first, index);
    uint32_t next = tile_page<TP>(c, src, min(first + 1, end - 1), index);
    load(first, page);
    stage(first, first, page);
    page = next;
    next = tile_page<TP>(c, src, min(first + 2, end - 1), index);
    load(min(first + 1, end - 1), page);
    __syncthreads();

    const auto scores = [&](uint32_t buf, f32x4 (&s)[QT][kTiles]) __attribute__((always_inline)) {
#pragma unroll
        for (int step = 0; step < NS; ++step) {
            const uint16_t *const ks = sh.k[buf] + piece_at<HD>(n, g * (HD / 32) + step);
            bf16x8 kf[kTiles];
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                kf[i] = *reinterpret_cast<const bf16x8 *>(ks + 16 * i * HD);
            }
#pragma unroll
            for (int p = QP - 1; p >= 0; --p) {
#pragma unroll
                for (uint32_t i = 0; i < kTiles; ++i) {
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi) {
                        s[qi][i] = mf::mfma(kf[i], qf[qi][step][p],
                                            step == 0 && p == QP - 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[qi][i]);
                    }
                }
            }
        }
    };
    const auto soften = [&](uint32_t chunk, f32x4 (&s)[QT][kTiles]) __attribute__((always_inline)) {
        softmax_step<HD, M>(s, st, mine, whole.has(chunk), int32_t(chunk * kChunk + 4 * g), a.c);
    };
#pragma unroll 1
    for (uint32_t chunk = first; chunk < end; ++chunk) {
        const uint32_t buf = chunk % 2;
        f32x4 s[QT][kTiles];
        if (needed.has(chunk)) {
            scores(buf, s);
        }
        // the next chunk into the other buffer, whose readers are behind the last barrier (at the
        // end the last one again, which nobody reads)
        stage(chunk + 1, min(chunk + 1, end - 1), page);
        page = next;
        next = tile_page<TP>(c, src, min(chunk + 3, end - 1), index);
        load(min(chunk + 2, end - 1), page);
        if (needed.has(chunk)) {
            soften(chunk, s);
            weigh_values<HD, PP, M>(sh.v[buf], s, st, n, g);
            const uint32_t some = uint32_t(sh.nans[buf][0] | sh.nans[buf][1]) |
                                  uint32_t(sh.nans[buf][2] | sh.nans[buf][3]);
            if (__builtin_amdgcn_readfirstlane(some)) {
#pragma unroll 1
                for (uint32_t i = 0; i < kTiles; ++i) {
                    if (!sh.nans[buf][i]) {
                        continue;  // (nothing was noted of its positions)
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t local = 16 * i + 4 * g + j;
                        const int32_t p = int32_t(chunk * kChunk + local);
                        const uint32_t bits = sh.nan[buf][local];
#pragma unroll
                        for (int qi = 0; qi < QT; ++qi) {
                            nan_blocks[qi] |= p >= mine[qi].first && p <= mine[qi].last ? bits : 0u;
                        }
                    }
                }
            }
        }
        __syncthreads();
    }

#pragma unroll
    for (int qi = 0; qi < QT; ++qi) {
        const uint32_t query = own + 16 * qi + n, token = query / a.group;
        const uint32_t poison = or_over_groups(nan_blocks[qi]);
        const float l = sum_over_groups(st.l[qi]);
        if (query >= limit) {
            continue;
        }
        const uint32_t head = kv_head * a.group + query - token * a.group;
        const bool idle = k.position0 + int32_t(token) < 0;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            f32x4 o = st.o[qi][mt];
            if (poison >> (mt / 2) & 1) {
                o = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
            const uint32_t d = 16 * mt + 4 * g;
            if (place < 0) {
                store4(out + (size_t(k.row0 + token) * a.heads + head) * HD + d,
                       idle ? f32x4{0.f, 0.f, 0.f, 0.f} : with_sink(a, head, st.b[qi], o, l));
            } else {
                const size_t to_place =
                    ((size_t(kv_head) * plan.shares + share) * 2 + uint32_t(place)) * plan.queries + (query - k.query0);
                *reinterpret_cast<f32x4 *>(plan.o + to_place * HD + d) = o;
                if (d == 0) {
                    plan.bl[to_place] = make_float2(st.b[qi], l);
                }
            }
        }
    }
}

template <int HD, class T, int TP>
__global__ __launch_bounds__((Tile<HD, T>::threads))
    __attribute__((amdgpu_waves_per_eu(Tile<HD, T>::waves_per_simd))) void
attention_tile_kernel(Cache c, Batch b, Params a, Plan plan, const T *__restrict__ q, T *__restrict__ out) {
    __shared__ __attribute__((aligned(16))) TileShared<HD, T> sh;
    do_share<HD, T, Tile<HD, T>::waves>(
        b, a, plan, sh.scan, out, [&](const Block &k, uint32_t from, uint32_t to, int place) {
            do_tile<HD, T, TP>(c, b, a, plan, k, blockIdx.y, from, to, place, blockIdx.x, sh, q, out);
        });
}

// ---- the parts of a block joined ---------------------------------------------------------------

// W waves per row and head, P parts at a time each (HD / 4 lanes a part): 4 waves where few
// rows may have many parts; one where rows are few; else only the lanes of one part (P = 1),
// which takes fewer waves for what is mostly waiting.  In us with the attention, for W, P = 4 and
// all, 1 and all, 1 and 1: 64 rows of 96 parts (one token at 131072) 26.8, 28.1, 26.8; 64 rows of 9
// parts 10.9, 11.1, 12.3; 2048 rows (4 tokens of 8 sequences at 16384) 39, 37.8, 40; 4096 rows (64
// ragged sequences) 54.3, 50.6, 50.8; 32768 rows (512 tokens at 2048) 107, 79, 71.
template <int HD, class T, int W, int P>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(Cache c, Batch b, Params a, Plan plan,
                                                                  T *__restrict__ out) {
    constexpr uint32_t kLanes = HD / 4, kSpan = P * kLanes, kRows = 64 / kSpan;  // rows (and heads) of a wave
    __shared__ float part_l[kWaves];
    __shared__ f32x4 part_o[kWaves][kLanes];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % kSpan;
    const uint32_t at = (blockIdx.x * (kWaves / W) + wave / W) * kRows + threadIdx.x % 64 / kSpan, turn = wave % W;
    const uint32_t row = at / a.heads, head = at % a.heads, kv_head = head / a.group;
    const uint32_t part = lane / kLanes, d = 4 * (lane % kLanes);
    T *const dst = out + (size_t(row) * a.heads + head) * HD + d;
    uint32_t parts = 0, first = 0, local = 0;
    if (row < b.tokens) {
        const kv4::Row r = kv4::row_of(b, row);
        if (r.kind == kv4::kToken) {
            const uint32_t row0 = b.starts ? uint32_t(max(kv4::entry(b.starts, r.sequence), 0)) : r.sequence;
            const uint32_t query = (row - row0) * a.group + head % a.group;
            local = query % plan.queries;
            const uint32_t block = b.starts ? uint32_t(uint64_t(row0) * a.group / plan.queries) + r.sequence
                                            : r.sequence * ((a.group + plan.queries - 1) / plan.queries);
            const uint2 span = plan.span[block + query / plan.queries];
            // (bounded, so that starts out of order cannot lead out of the workspace)
            first = min(span.x, plan.shares - 1);
            parts = min(span.y - first, plan.shares - 1 - first) + 1;
        } else if (r.kind != kv4::kPadding && turn == 0 && part == 0) {
            const float fill = r.kind == kv4::kBad ? __builtin_nanf("") : 0.0f;
            store4(dst, f32x4{fill, fill, fill, fill});
        }
    }
    if (W == 1 && parts <= 1) {
        return;  // (one part: the workgroup that had it wrote the output)
    }
    const auto place = [&](uint32_t i) {
        return ((size_t(kv_head) * plan.shares + first + i) * 2 + (i == 0 ? 1 : 0)) * plan.queries + local;
    };
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, l = 0.0f;
    if (parts > 1) {
        for (uint32_t i = lane; i < parts; i += kSpan) {
            top = fmaxf(top, plan.bl[place(i)].x);
        }
#pragma unroll
        for (int x = kSpan / 2; x >= 1; x >>= 1) {
            top = fmaxf(top, __shfl_xor(top, x));
        }
        const float offset = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
        for (uint32_t i = turn * P + part; i < parts; i += W * P) {
            const float2 s = plan.bl[place(i)];
            const f32x4 x = *reinterpret_cast<const f32x4 *>(plan.o + place(i) * HD + d);
            const float f = __builtin_amdgcn_exp2f(s.x - offset);
            l = fmaf(s.y, f, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = fmaf(x[j], f, o[j]);
            }
        }
#pragma unroll
        for (uint32_t x = kLanes; x < kSpan; x <<= 1) {
            l += __shfl_xor(l, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] += __shfl_xor(o[j], x);
            }
        }
    }
    if (W > 1) {
        if (part == 0) {
            part_o[wave][lane] = o;
            part_l[wave] = l;
        }
        __syncthreads();
        if (turn != 0 || parts <= 1) {
            return;
        }
#pragma unroll
        for (uint32_t x = 1; x < W; ++x) {
            l += part_l[wave + x];
            const f32x4 y = part_o[wave + x][lane % kLanes];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] += y[j];
            }
        }
    }
    if (part == 0) {
        store4(dst, with_sink(a, head, top, o, l));
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

template <int M>
uint32_t resident_groups(uint32_t head_dim, int dtype) {
    const bool f32 = dtype == TTL_DTYPE_F32;
    return head_dim == 64 ? (f32 ? kResident<64, float, M> : kResident<64, __bf16, M>)
                          : (f32 ? kResident<128, float, M> : kResident<128, __bf16, M>);
}

// The cut of a checked call, by the queries that a sequence has on average: few share a
// workgroup's waves, from kTileFrom on each wave has its own.  Heads of 64 over long contexts
// fill a wave with less: from kTileFromLong on where a query sees more than kLongChunks (64
// sequences of 128 queries, bf16: at 2048 the split kernel takes 108 against 146 us, with a window
// of 128 43 against 36; of 192 queries at 1024 103 against 87, 8 of 256 at 4096 49 against 53, 64
// of 256 with the window 78 against 45; heads of 128, 8 sequences of 200 queries at 4096: 55
// against 48).  What a query sees goes by max_length, the bound that the call states.
struct Cut {
    bool tile;
    int mode;
    Plan plan;
    uint32_t most_parts;  // of a block
    size_t workspace;
};
constexpr uint64_t kTileFrom = 64, kTileFromLong = 256;
constexpr uint32_t kLongChunks = 24, kShortChunks = 8;
constexpr uint64_t kCus = 256;
Cut cut_of(const ttl_kv4_cache *cache, const ttl_kv4_batch *batch, const ttl_kv4_attention *attention) {
    const uint32_t group = attention->heads / cache->kv_heads;
    const bool f32 = attention->dtype == TTL_DTYPE_F32;
    Cut cut{};
    const uint64_t queries = uint64_t(batch->tokens) * group;  // of a key/value head
    const uint64_t mean = queries / batch->sequences;
    Plan &p = cut.plan;
    const uint64_t seen = attention->window
                              ? std::min<uint64_t>(batch->max_length, uint64_t(attention->window) + mean / group)
                              : batch->max_length;
    const bool fits = cache->head_dim == 64 && seen / kChunk > kLongChunks;
    cut.tile = batch->starts && mean >= (fits ? kTileFromLong : kTileFrom);
    uint64_t slots = 0;
    if (cut.tile) {
        const auto take = [&](auto tile) {
            p.queries = decltype(tile)::queries;
            slots = kCus * decltype(tile)::groups;
        };
        if (cache->head_dim == 64) {
            f32 ? take(Tile<64, float>()) : take(Tile<64, __bf16>());
        } else {
            f32 ? take(Tile<128, float>()) : take(Tile<128, __bf16>());
        }
        p.unit = 1;
    } else {
        cut.mode = mean > 16 ? kTwo : mean > 8 ? kOne : kHalf;
        p.queries = cut.mode == kTwo ? 32 : cut.mode == kOne ? 16 : 8;
        p.unit = kWaves;
        slots = kCus * (cut.mode == kHalf  ? resident_groups<kHalf>(cache->head_dim, attention->dtype)
                        : cut.mode == kOne ? resident_groups<kOne>(cache->head_dim, attention->dtype)
                                           : resident_groups<kTwo>(cache->head_dim, attention->dtype));
    }
    p.blocks = batch->starts ? uint32_t(queries / p.queries + batch->sequences)
                             : batch->sequences * ((group + p.queries - 1) / p.queries);
    uint32_t longest = batch->max_length;
    if (attention->window) {
        // a block's tokens span queries / group + 1 positions at most
        longest = uint32_t(std::min<uint64_t>(longest, uint64_t(attention->window) + p.queries / group + 1));
    }
    const uint32_t chunks = longest / kChunk + (attention->window ? 2 : 1);  // any alignment
    const uint64_t units = (chunks + p.unit - 1) / p.unit;
    // A workgroup takes a block whole where blocks are enough (1024 tokens at 2048: 75 against 83
    // us), or short enough for half as many (4 x 128 tokens at 1024: 41 against 43 us; but 512 at
    // 8192: 238 against 144), or so short that the join costs more than a workgroup's walk (a
    // prompt of 300: 14 against 22 us; two of 100 at 1400, f32: 51 against 40), or so many that
    // finding a share would take long, the units pass 31 bits or the join a grid.  Blocks are as long
    // as max_length lets them be: under a bound of 131072 a prompt of 300 is divided.
    const uint64_t all = uint64_t(p.blocks) * cache->kv_heads;
    const bool whole = all >= slots || (2 * all >= slots && units <= kLongChunks) || units <= kShortChunks;
    p.single = units == 1 || (cut.tile && whole) || p.blocks > 1u << 16 || p.blocks * units > 1u << 31 ||
               uint64_t(batch->tokens) * attention->heads > 1u << 26;
    if (p.single) {
        p.shares = p.blocks;
        return cut;
    }
    p.shares = uint32_t(std::max<uint64_t>(1, slots / cache->kv_heads));
    p.shares = uint32_t(std::min<uint64_t>(p.shares, units * p.blocks));
    // a block spans the shares of its units
    cut.most_parts = uint32_t(std::min<uint64_t>(p.shares, units + 1));
    const size_t places = size_t(cache->kv_heads) * p.shares * 2 * p.queries;
    cut.workspace = places * (cache->head_dim * sizeof(float) + sizeof(float2)) + size_t(p.blocks) * sizeof(uint2);
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
    TTL_REQUIRE(uint64_t(cut.plan.shares) * 2 * kThreads <= 0xffffffffu &&  // (a launch's threads)
                    uint64_t(batch->tokens) * attention->heads <= 0x7fffffffu,
                TTL_ERR_SHAPE,
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
    if (!p.single) {
        const size_t places = size_t(cache->kv_heads) * p.shares * 2 * p.queries;
        p.o = static_cast<float *>(workspace);
        p.bl = reinterpret_cast<float2 *>(p.o + places * cache->head_dim);
        p.span = reinterpret_cast<uint2 *>(p.bl + places);
    }
    const auto launch = [&](auto hd, auto zero) {
        constexpr int HD = decltype(hd)::value;
        using T = decltype(zero);
        const T *qt = static_cast<const T *>(q);
        T *ot = static_cast<T *>(out);
        const dim3 grid(p.shares, c.kv_heads);
        const bool big = c.page_shift >= 6;
        const auto split = [&](auto mode) {
            constexpr int M = decltype(mode)::value;
            if (big) {
                attention_split_kernel<HD, T, M, 1><<<grid, kThreads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            } else {
                attention_split_kernel<HD, T, M, 4><<<grid, kThreads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            }
        };
        if (cut.tile) {
            constexpr uint32_t threads = Tile<HD, T>::threads;
            if (big) {
                attention_tile_kernel<HD, T, 1><<<grid, threads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            } else {
                attention_tile_kernel<HD, T, 4><<<grid, threads, 0, ctx->stream>>>(c, b, a, p, qt, ot);
            }
        } else if (cut.mode == kHalf) {
            split(std::integral_constant<int, kHalf>());
        } else if (cut.mode == kOne) {
            split(std::integral_constant<int, kOne>());
        } else {
            split(std::integral_constant<int, kTwo>());
        }
        if (!p.single) {
            const size_t rows = size_t(b.tokens) * a.heads;
            constexpr int P = 256 / HD;
            if (cut.most_parts > 16 && rows <= 1024) {
                attention_join_kernel<HD, T, 4, P><<<uint32_t(rows), kThreads, 0, ctx->stream>>>(c, b, a, p, ot);
            } else if (rows <= 4096) {
                attention_join_kernel<HD, T, 1, P><<<ttl::blocks_for(rows, kWaves), kThreads, 0, ctx->stream>>>(
                    c, b, a, p, ot);
            } else {
                attention_join_kernel<HD, T, 1, 1><<<ttl::blocks_for(rows, kWaves * P), kThreads, 0, ctx->stream>>>(
                    c, b, a, p, ot);
            }
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
