// Decode kernels over a KV pool held in 4 bits, gfx950 (CDNA4, 64-lane wavefronts), head_size = value_size = 64, 128, 192 or
// 256.
//
// A wavefront takes the up to 16 query heads of one KV head together and walks a run of tokens in steps of 32 (two tiles of
// 16), so that every byte of the pool is read once. lane = 16 g + c (g = 0..3, c = 0..15). Per tile:
//   S[token][head] = K . Q^T   v_mfma_f32_16x16x32, A = K: lane c holds HEAD / 4 neighbouring elements of one token, straight
//                              from the load. The matrix instruction sums over the elements whatever their order, as long as
//                              the query has the same, so a lane's elements need not be spread over the four groups g, and
//                              each lane's codes lie under one scale (two above head 128).
//   O[head][dim] += P . V      v_mfma_f32_16x16x32 over both tiles of a step, A = P as S came out, B = V: the lane that loads
//                              a strip of columns of tokens 4 i + g (i = 0..3) is the lane that feeds those to the matrix
//                              unit; pairs of tokens are interleaved with byte permutes.
// So nothing passes through LDS. Row m of a tile is token 4 (m % 4) + m / 4: the accumulator rows of group g are then tokens
// g, 4 + g, 8 + g, 12 + g, and each V load instruction covers four neighbouring rows.
//
// Codes become bf16 or fp16 under their scale by v_cvt_scalef32_pk_*, two elements per instruction: K in the query's type, V
// in fp16, where every written value is exact and the probabilities keep eleven bits (as bf16 they would add an error as large
// as the output's own rounding). For fp16 outputs the probabilities go in as two terms for the same reason.
//
// Work is dealt by steps: the steps of all sequences, one after the other, are cut into as many equal runs as there are
// wavefronts for a KV head. A run may hold the end of one sequence, whole ones, and the start of another; whole sequences are
// normalised and written at once, the others leave accumulators, reference points and denominators, which the merge kernel
// joins in the order of the runs.
#ifndef INFINICORE_AMD_PA_DECODE_FP4_H
#define INFINICORE_AMD_PA_DECODE_FP4_H

#include "../../../devices/amd/amd_fp4.h"
#include "../../paged_attention/amd/decode_tiled.h"

namespace op::paged_attention_fp4::amd {

using op::paged_attention::amd::BFloat16;
using op::paged_attention::amd::clampPage;
using op::paged_attention::amd::f32x4;
using op::paged_attention::amd::fastExp2;
using op::paged_attention::amd::Half;
using op::paged_attention::amd::kHeadsPerWave;
using op::paged_attention::amd::kLog2e;
using op::paged_attention::amd::maxAcrossTokenGroups;
using op::paged_attention::amd::maxOf;
using op::paged_attention::amd::sumAcrossTokenGroups;
using op::paged_attention::amd::TileBF16;
using op::paged_attention::amd::TileF16;
using op::paged_attention::amd::waveInclusiveSum;
namespace mx = device::amd::mx;

constexpr int kStepTokens = 32;
constexpr int kDecodeThreads = 256;  // four wavefronts that share nothing but the launch
constexpr int kLeastSteps = 4;       // of a run: below that the merge costs more than it saves
constexpr float kLazyLog2 = 8.0f;    // how far (in powers of two) a maximum may outgrow its reference point

enum class IndexType : int32_t { i64, i32, u32 };

__device__ __forceinline__ int64_t loadIndexOf(IndexType type, const void *base, int64_t i) {
    if (type == IndexType::i64) {
        return static_cast<const int64_t *>(base)[i];
    }
    return type == IndexType::i32 ? static_cast<int64_t>(static_cast<const int32_t *>(base)[i])
                                  : static_cast<int64_t>(static_cast<const uint32_t *>(base)[i]);
}

// One of the pool's tensors; strides in bytes.
struct PoolSide {
    const char *base;
    int64_t block, head;
    int32_t row;
};

struct DecodeFp4Args {
    void *out;
    const void *q;
    PoolSide k_codes, k_scales, v_codes, v_scales;
    const void *block_tables;
    const void *seq_lens;
    const float *alibi_slopes; // nullptr = no ALiBi
    IndexType index_type;

    // partial results, two places per run: [stream][run][0 = of a sequence that began before it, 1 = of one that ends behind it]
    float *part_acc;  // [..][part_rows][HEAD]
    float2 *part_ml;  // [..][part_rows] reference point (log2), denominator
    int32_t part_rows; // heads of a chunk: min(group, 16)

    float scale_log2; // scale * log2(e)
    int32_t num_seqs, num_heads, num_kv_heads;
    int32_t group;       // query heads per KV head
    int32_t head_chunks; // of up to 16 query heads
    int32_t runs;        // per stream (KV head and chunk), at most
    int32_t block_size;
    int32_t num_blocks;  // pool size; table entries are clamped into [0, num_blocks)
    int32_t capacity;    // tokens that a row of the block table can hold, at most
    bool q_aligned;      // every query row begins at a multiple of 16 bytes
    bool out_aligned;    // and every output row
    int64_t q_stride, q_head_stride; // elements
    int64_t o_stride, o_head_stride;
    int64_t block_table_stride;
};

// Tokens of sequence `seq`, forced into what its table can hold.
__device__ __forceinline__ int sequenceTokens(const DecodeFp4Args &a, int seq) {
    const int64_t n = loadIndexOf(a.index_type, a.seq_lens, seq);
    return static_cast<int>(n < 0 ? 0 : (n > a.capacity ? a.capacity : n));
}
__device__ __forceinline__ int stepsOf(int tokens) { return (tokens + kStepTokens - 1) / kStepTokens; }

// The runs that `steps` steps are cut into: run i has steps [i steps / runs, (i + 1) steps / runs).
__device__ __forceinline__ int runsFor(const DecodeFp4Args &a, int64_t steps) {
    const int64_t most = (steps + kLeastSteps - 1) / kLeastSteps;
    return static_cast<int>(most < a.runs ? most : a.runs);
}
__device__ __forceinline__ int64_t runStart(int64_t steps, int runs, int run) { return steps * run / runs; }
__device__ __forceinline__ int runOf(int64_t steps, int runs, int64_t step) { return static_cast<int>(((step + 1) * runs - 1) / steps); }

// Steps of all sequences.
__device__ __forceinline__ int64_t totalSteps(const DecodeFp4Args &a, int lane) {
    int64_t total = 0;
    for (int base = 0; base < a.num_seqs; base += 64) {
        const int n = base + lane < a.num_seqs ? stepsOf(sequenceTokens(a, base + lane)) : 0;
        total += __builtin_amdgcn_readlane(waveInclusiveSum(n), 63);
    }
    return total;
}

template <int BYTES> struct Bits;
template <> struct Bits<2> { using type = uint16_t; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<8> { typedef unsigned type __attribute__((ext_vector_type(2))); };
template <> struct Bits<16> { typedef unsigned type __attribute__((ext_vector_type(4))); };
// ONCE: past the caches, for what a call reads once.
template <int BYTES, bool ONCE = true>
__device__ __forceinline__ void loadWords(const char *p, uint32_t *to) {
    const auto *from = reinterpret_cast<const typename Bits<BYTES>::type *>(p);
    const auto v = ONCE ? __builtin_nontemporal_load(from) : *from;
    if constexpr (BYTES <= 4) {
        to[0] = v;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) {
            to[i] = v[i];
        }
    }
}

// How a head's elements and columns lie in the lanes. K: pieces of 128 (32 elements a lane, one 16-byte load) and, at 64
// and 192, one of 64 (16 elements, 8 bytes). V: one strip of HEAD / 16 neighbouring columns a lane, at head 192 a strip of
// 8 columns out of the first 128 and one of 4 out of the rest, so that no lane reads three bytes of two words.
template <int HEAD>
struct Layout {
    static constexpr int kWords = HEAD / 32;                   // dwords of K codes a lane and token
    static constexpr int kPieces = (HEAD + 127) / 128;         // of K
    static constexpr int kStrips = HEAD == 192 ? 2 : 1;        // of V
    static constexpr int kStripCols = HEAD == 192 ? 8 : HEAD / 16; // of the first
    static constexpr int kCols = HEAD / 16;
    static constexpr int kVWords = HEAD == 64 || HEAD == 128 ? 1 : 2;
    static constexpr bool pieceWhole(int p) { return 128 * p + 128 <= HEAD; }
    // first element and scale of lane group g in piece p
    static __device__ __forceinline__ int element(int p, int g) { return 128 * p + (pieceWhole(p) ? 32 : 16) * g; }
    // first column of lane c in strip s
    static __device__ __forceinline__ int column(int s, int c) { return s == 0 ? kStripCols * c : 128 + 4 * c; }
};

// What a lane loads of one step.
template <int HEAD>
struct Step {
    using L = Layout<HEAD>;
    uint32_t k[2][L::kWords];
    uint8_t ks[2][L::kPieces];
    uint32_t v[8][L::kVWords]; // [tile][i]: token 4 i + g
    uint8_t vs[8][L::kStrips];
};

// Where the rows of a sequence lie. GRAIN: the page size is a multiple of this many tokens; 16 = a tile lies in one page, 8 =
// each half of it does, 1 = every lane looks its rows up for itself.
template <int HEAD, int GRAIN>
struct Pages {
    using L = Layout<HEAD>;
    const DecodeFp4Args &a;
    int lane, g, c, kv_head;
    int64_t table;  // index of the sequence's first table entry
    int tokens;     // of the sequence
    // GRAIN > 1: the pages of 64 table entries, one a lane, and the unit (GRAIN tokens) that comes next
    int32_t ids;
    int first_entry, entry, row, token;

    __device__ __forceinline__ int32_t page(int64_t at) const {
        return clampPage(loadIndexOf(a.index_type, a.block_tables, table + at), a.num_blocks);
    }
    __device__ __forceinline__ void fetch(int from) {
        first_entry = from;
        const int last = (tokens - 1) / a.block_size;
        ids = page(min(from + lane, last));
    }
    __device__ __forceinline__ void begin(int seq, int tokens_, int step) {
        table = seq * a.block_table_stride;
        tokens = tokens_;
        token = step * kStepTokens;
        if constexpr (GRAIN > 1) {
            entry = token / a.block_size;
            row = token - entry * a.block_size;
            fetch(entry);
        }
    }
    static __device__ __forceinline__ const char *rowOf(const PoolSide &s, int32_t page, int kv_head, int row) {
        return s.base + page * s.block + kv_head * s.head + static_cast<int64_t>(row) * s.row;
    }

    struct Unit {
        const char *kc, *ks, *vc, *vs;
    };
    // The next GRAIN tokens; where the sequence has none left, the last ones again.
    __device__ __forceinline__ Unit next() {
        if (entry - first_entry >= 64) {
            fetch(entry);
        }
        const int32_t id = __builtin_amdgcn_readlane(ids, entry - first_entry);
        const Unit u{rowOf(a.k_codes, id, kv_head, row), rowOf(a.k_scales, id, kv_head, row), rowOf(a.v_codes, id, kv_head, row),
                     rowOf(a.v_scales, id, kv_head, row)};
        token += GRAIN;
        if (token < tokens) {
            row += GRAIN;
            if (row >= a.block_size) {
                row = 0;
                ++entry;
            }
        }
        return u;
    }

    __device__ __forceinline__ void loadK(Step<HEAD> &to, int tile, const char *codes, const char *scales) const {
#pragma unroll
        for (int p = 0; p < L::kPieces; ++p) {
            const int e = L::element(p, g);
            if (L::pieceWhole(p)) {
                loadWords<16>(codes + e / 2, &to.k[tile][4 * p]);
            } else {
                loadWords<8>(codes + e / 2, &to.k[tile][4 * p]);
            }
            to.ks[tile][p] = __builtin_nontemporal_load(reinterpret_cast<const uint8_t *>(scales + e / 32));
        }
    }
    __device__ __forceinline__ void loadV(Step<HEAD> &to, int at, const char *codes, const char *scales) const {
#pragma unroll
        for (int s = 0; s < L::kStrips; ++s) {
            const int d = L::column(s, c);
            if (s == 0) {
                loadWords<L::kStripCols / 2>(codes + d / 2, to.v[at]);
            } else {
                loadWords<2>(codes + d / 2, &to.v[at][1]);
            }
            to.vs[at][s] = __builtin_nontemporal_load(reinterpret_cast<const uint8_t *>(scales + d / 32));
        }
    }

    // The 32 tokens that come next.
    __device__ __forceinline__ void load(Step<HEAD> &to) {
        const int m = 4 * (c & 3) + (c >> 2); // this lane's K row of a tile
        if constexpr (GRAIN == 16) {
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                const Unit u = next();
                loadK(to, tile, u.kc + m * a.k_codes.row, u.ks + m * a.k_scales.row);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    loadV(to, 4 * tile + i, u.vc + 4 * i * a.v_codes.row + g * a.v_codes.row,
                          u.vs + 4 * i * a.v_scales.row + g * a.v_scales.row);
                }
            }
        } else if constexpr (GRAIN == 8) {
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                const Unit u = next(), w = next();
                const bool second = m >= 8;
                loadK(to, tile, (second ? w.kc : u.kc) + (m & 7) * a.k_codes.row, (second ? w.ks : u.ks) + (m & 7) * a.k_scales.row);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const Unit &x = i < 2 ? u : w;
                    const int r = 4 * (i & 1) + g;
                    loadV(to, 4 * tile + i, x.vc + r * a.v_codes.row, x.vs + r * a.v_scales.row);
                }
            }
        } else {
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                auto place = [&](int t, int32_t &id, int &r) {
                    t = min(t, tokens - 1);
                    const int e = t / a.block_size;
                    r = t - e * a.block_size;
                    id = page(e);
                };
                int32_t id;
                int r;
                place(token + 16 * tile + m, id, r);
                loadK(to, tile, rowOf(a.k_codes, id, kv_head, r), rowOf(a.k_scales, id, kv_head, r));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    place(token + 16 * tile + 4 * i + g, id, r);
                    loadV(to, 4 * tile + i, rowOf(a.v_codes, id, kv_head, r), rowOf(a.v_scales, id, kv_head, r));
                }
            }
            token += kStepTokens;
        }
    }
};

template <typename T, int HEAD>
struct DecodeState {
    uint4 q[HEAD / 32];
    f32x4 o[HEAD / 16];
    float m, l; // of head c: reference point of the exponentials (log2), this lane's part of the denominator
};

template <typename T>
__device__ __forceinline__ uint4 toQueryType(uint32_t codes, float scale);
template <>
__device__ __forceinline__ uint4 toQueryType<TileBF16>(uint32_t codes, float scale) { return mx::toBF16x8(codes, scale); }
template <>
__device__ __forceinline__ uint4 toQueryType<TileF16>(uint32_t codes, float scale) { return mx::toF16x8(codes, scale); }

// Columns 2 B and 2 B + 1 of a strip: the operands of eight tokens each.
template <int B, int HEAD>
__device__ __forceinline__ void columnPair(const Step<HEAD> &s, const float (&scale)[8], int word, uint4 &even, uint4 &odd) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = mx::toF16<B>(s.v[j][word], scale[j]);
    }
    auto low = [](uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x05040100u); };
    auto high = [](uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); };
    even = make_uint4(low(w[0], w[1]), low(w[2], w[3]), low(w[4], w[5]), low(w[6], w[7]));
    odd = make_uint4(high(w[0], w[1]), high(w[2], w[3]), high(w[4], w[5]), high(w[6], w[7]));
}

// One step. Tokens from `left` on are behind the sequence; what their rows hold has no part in anything.
template <typename T, int HEAD>
__device__ __forceinline__ void computeStep(const DecodeFp4Args &a, const Step<HEAD> &s, DecodeState<T, HEAD> &st, int g, int left,
                                            float slope_log2, float away) {
    using L = Layout<HEAD>;
    constexpr bool kSplit = T::kSplitProbabilities == false; // fp16 outputs: two terms (see the top)
    f32x4 score[2];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < L::kWords; ++w) {
            x = T::mfmaK32(toQueryType<T>(s.k[tile][w], mx::scaleOf(s.ks[tile][w / 4])), st.q[w], x);
        }
        score[tile] = x * a.scale_log2;
    }
    if (a.alibi_slopes != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            score[j / 4][j & 3] += slope_log2 * (away + static_cast<float>(16 * (j / 4) + 4 * (j & 3) + g));
        }
    }
    if (left < kStepTokens) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            score[j / 4][j & 3] = 16 * (j / 4) + 4 * (j & 3) + g < left ? score[j / 4][j & 3] : -INFINITY;
        }
    }
    const float top = maxOf(maxOf(maxOf(score[0][0], score[0][1]), maxOf(score[0][2], score[0][3])),
                            maxOf(maxOf(score[1][0], score[1][1]), maxOf(score[1][2], score[1][3])));
    // (a NaN compares as not greater; it reaches the outputs by its own probability)
    if (__builtin_amdgcn_ballot_w64(top > st.m + kLazyLog2) != 0) {
        const float m = maxOf(st.m, maxAcrossTokenGroups(top));
        const float alpha = st.m == m ? 1.0f : fastExp2(st.m - m);
        st.l *= alpha;
        st.m = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = __shfl(alpha, 4 * g + i, 64);
#pragma unroll
            for (int e = 0; e < L::kCols; ++e) {
                st.o[e][i] *= f;
            }
        }
    }
    float p[8];
    const float from = st.m == -INFINITY ? 0.0f : st.m; // products that overflowed, all of them so far: no weight, not a NaN
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = fastExp2(score[j / 4][j & 3] - from);
    }
    st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    const uint4 hi = make_uint4(TileF16::pack2(p[0], p[1]), TileF16::pack2(p[2], p[3]), TileF16::pack2(p[4], p[5]),
                                TileF16::pack2(p[6], p[7]));
    uint4 lo = make_uint4(0, 0, 0, 0);
    if constexpr (kSplit) {
        auto rest = [](float x, float y, uint32_t w) { return TileF16::pack2(x - TileF16::unpackLo(w), y - TileF16::unpackHi(w)); };
        lo = make_uint4(rest(p[0], p[1], hi.x), rest(p[2], p[3], hi.y), rest(p[4], p[5], hi.z), rest(p[6], p[7], hi.w));
    }

#pragma unroll
    for (int strip = 0; strip < L::kStrips; ++strip) {
        float scale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            scale[j] = mx::scaleOf(s.vs[j][strip]);
        }
        if (left < kStepTokens) { // a NaN there would pass through a probability of zero
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                scale[j] = 16 * (j / 4) + 4 * (j & 3) + g < left ? scale[j] : 0.0f;
            }
        }
        constexpr int kFirst = L::kStripCols;
        auto pair = [&](auto at, int word, int column) {
            uint4 even, odd;
            columnPair<decltype(at)::value, HEAD>(s, scale, word, even, odd);
            st.o[column] = TileF16::mfmaK32(hi, even, st.o[column]);
            st.o[column + 1] = TileF16::mfmaK32(hi, odd, st.o[column + 1]);
            if constexpr (kSplit) {
                st.o[column] = TileF16::mfmaK32(lo, even, st.o[column]);
                st.o[column + 1] = TileF16::mfmaK32(lo, odd, st.o[column + 1]);
            }
            if constexpr (HEAD > 128) {
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto word = [&](int w, int column, auto cols) {
            pair(std::integral_constant<int, 0>{}, w, column);
            pair(std::integral_constant<int, 1>{}, w, column + 2);
            if constexpr (decltype(cols)::value == 8) {
                pair(std::integral_constant<int, 2>{}, w, column + 4);
                pair(std::integral_constant<int, 3>{}, w, column + 6);
            }
        };
        if (strip == 0) {
            word(0, 0, std::integral_constant<int, (kFirst < 8 ? 4 : 8)>{});
            if constexpr (kFirst == 16) {
                word(1, 8, std::integral_constant<int, 8>{});
            }
        } else {
            word(1, 8, std::integral_constant<int, 4>{});
        }
    }
}

// The query heads of a chunk of sequence `seq`, in the order of the K elements; heads that the chunk does not have as zeros.
template <typename T, int HEAD>
__device__ __forceinline__ void loadQuery(const DecodeFp4Args &a, int seq, int kv_head, int chunk, int g, int c, uint4 (&q)[HEAD / 32]) {
    using L = Layout<HEAD>;
    using S = typename T::storage;
    const int h = chunk * kHeadsPerWave + c;
    const S *row = static_cast<const S *>(a.q) + seq * a.q_stride + (kv_head * a.group + min(h, a.group - 1)) * a.q_head_stride;
#pragma unroll
    for (int w = 0; w < L::kWords; ++w) {
        const S *at = row + L::element(w / 4, g) + 8 * (w & 3);
        uint4 x;
        if (a.q_aligned) {
            x = *reinterpret_cast<const uint4 *>(at);
        } else {
            const uint16_t *e = reinterpret_cast<const uint16_t *>(at);
            x = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
        q[w] = h < a.group ? x : make_uint4(0, 0, 0, 0);
    }
}

// The columns of strip s of one output row, rounded once.
template <typename T, int COLS>
__device__ __forceinline__ void storeColumns(typename T::storage *to, const float *x, bool aligned) {
    uint32_t w[COLS / 2];
#pragma unroll
    for (int i = 0; i < COLS / 2; ++i) {
        w[i] = T::pack2(x[2 * i], x[2 * i + 1]);
    }
    if (aligned) {
        if constexpr (COLS == 4) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < COLS / 8; ++i) {
                *reinterpret_cast<uint4 *>(to + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
            reinterpret_cast<uint16_t *>(to)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// What the lanes hold of a run of steps: normalised outputs (`whole`), or a partial result at place `place`.
template <typename T, int HEAD>
__device__ __forceinline__ void finish(const DecodeFp4Args &a, const DecodeState<T, HEAD> &st, bool whole, int64_t place, int seq,
                                       int kv_head, int chunk, int lane) {
    using L = Layout<HEAD>;
    const int g = lane >> 4, c = lane & 15;
    const float l = sumAcrossTokenGroups(st.l);
    const int heads = min(a.group - chunk * kHeadsPerWave, kHeadsPerWave);
    if (!whole && g == 0 && c < heads) {
        a.part_ml[place * a.part_rows + c] = make_float2(st.m, l);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int h = 4 * g + i;
        const float f = whole ? 1.0f / __shfl(l, h, 64) : 1.0f;
        if (h >= heads) {
            continue;
        }
        float x[L::kCols];
#pragma unroll
        for (int e = 0; e < L::kCols; ++e) {
            x[e] = st.o[e][i] * f;
        }
        if (whole) {
            auto *row = static_cast<typename T::storage *>(a.out) + seq * a.o_stride
                      + (kv_head * a.group + chunk * kHeadsPerWave + h) * a.o_head_stride;
            storeColumns<T, L::kStripCols>(row + L::column(0, c), x, a.out_aligned);
            if constexpr (L::kStrips > 1) {
                storeColumns<T, 4>(row + L::column(1, c), x + L::kStripCols, a.out_aligned);
            }
        } else {
            float *row = a.part_acc + (place * a.part_rows + h) * HEAD;
#pragma unroll
            for (int e = 0; e < L::kCols; e += 4) {
                const int strip = e < L::kStripCols ? 0 : 1;
                float *to = row + L::column(strip, c) + (strip == 0 ? e : e - L::kStripCols);
                *reinterpret_cast<float4 *>(to) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            }
        }
    }
}

template <typename T, int HEAD, int GRAIN>
__global__ void __launch_bounds__(kDecodeThreads, 2) decodeFp4Kernel(DecodeFp4Args a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int streams = a.num_kv_heads * a.head_chunks;
    const int stream = blockIdx.x % streams;
    const int run = static_cast<int>(blockIdx.x / streams) * (kDecodeThreads / 64) + wave;
    const int kv_head = stream / a.head_chunks, chunk = stream % a.head_chunks;

    const int64_t total = totalSteps(a, lane);
    const int runs = runsFor(a, total);
    if (run >= runs) {
        return;
    }
    int64_t at = runStart(total, runs, run);
    const int64_t end = runStart(total, runs, run + 1);

    const float slope = a.alibi_slopes != nullptr && chunk * kHeadsPerWave + c < a.group
                          ? a.alibi_slopes[kv_head * a.group + chunk * kHeadsPerWave + c] * kLog2e : 0.0f;
    Pages<HEAD, GRAIN> pages{a, lane, g, c, kv_head};
    DecodeState<T, HEAD> st;

    int64_t before = 0; // steps of the sequences in front of the 64 at hand
    for (int base = 0; base < a.num_seqs && at < end; base += 64) {
        const int tokens_of = base + lane < a.num_seqs ? sequenceTokens(a, base + lane) : 0;
        const int sum = waveInclusiveSum(stepsOf(tokens_of));
        const int all = __builtin_amdgcn_readlane(sum, 63);
        while (at < end && at < before + all) {
            // the first sequence that ends behind `at`
            const int in = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > at));
            const int tokens = __builtin_amdgcn_readlane(tokens_of, in);
            const int steps = stepsOf(tokens);
            const int64_t start = before + __builtin_amdgcn_readlane(sum, in) - steps;
            const int seq = base + in;
            const int from = static_cast<int>(at - start);
            const int to = static_cast<int>(end - start < steps ? end - start : steps);

            pages.begin(seq, tokens, from);
            Step<HEAD> ahead[2];
            pages.load(ahead[0]);
            loadQuery<T, HEAD>(a, seq, kv_head, chunk, g, c, st.q);
            st.m = -INFINITY;
            st.l = 0.0f;
#pragma unroll
            for (int e = 0; e < HEAD / 16; ++e) {
                st.o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            auto compute = [&](const Step<HEAD> &s, int step) {
                const int left = tokens - step * kStepTokens;
                // (1 - left: of the step's first token from the last one)
                computeStep<T, HEAD>(a, s, st, g, left, slope, static_cast<float>(1 - left));
            };
            for (int step = from; step < to; step += 2) {
                if (step + 1 < to) {
                    pages.load(ahead[1]);
                }
                compute(ahead[0], step);
                if (step + 1 < to) {
                    if (step + 2 < to) {
                        pages.load(ahead[0]);
                    }
                    compute(ahead[1], step + 1);
                }
            }
            const int64_t place = (static_cast<int64_t>(stream) * a.runs + run) * 2 + (from == 0 ? 1 : 0);
            finish<T, HEAD>(a, st, from == 0 && to == steps, place, seq, kv_head, chunk, lane);
            at = start + to;
        }
        before += all;
    }
}

// One wavefront per (sequence, query head): the parts of a sequence that lies in more than one run, joined in their order.
template <typename T, int HEAD>
__global__ void __launch_bounds__(64) mergeFp4Kernel(DecodeFp4Args a) {
    const int lane = threadIdx.x;
    const int seq = blockIdx.x / a.num_heads, head = blockIdx.x % a.num_heads;
    const int steps = stepsOf(sequenceTokens(a, seq));
    if (steps == 0) {
        return;
    }
    int64_t total = 0, start = 0;
    for (int base = 0; base < a.num_seqs; base += 64) {
        const int n = base + lane < a.num_seqs ? stepsOf(sequenceTokens(a, base + lane)) : 0;
        total += __builtin_amdgcn_readlane(waveInclusiveSum(n), 63);
        start += __builtin_amdgcn_readlane(waveInclusiveSum(base + lane < seq ? n : 0), 63);
    }
    const int runs = runsFor(a, total);
    const int first = runOf(total, runs, start), last = runOf(total, runs, start + steps - 1);
    if (first == last) {
        return; // whole: written already
    }
    const int kv_head = head / a.group, in_group = head % a.group;
    const int stream = kv_head * a.head_chunks + in_group / kHeadsPerWave;
    const int row = in_group % kHeadsPerWave;
    // a part is at place 1 where the sequence begins in that run, else at 0
    auto placeOf = [&](int run) {
        return ((static_cast<int64_t>(stream) * a.runs + run) * 2 + (run == first ? 1 : 0)) * a.part_rows + row;
    };
    float m = -INFINITY;
    for (int run = first + lane; run <= last; run += 64) {
        m = maxOf(m, a.part_ml[placeOf(run)].x);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        m = maxOf(m, __shfl_xor(m, off, 64));
    }
    constexpr int kPer = HEAD / 64;
    float l = 0.0f, x[kPer] = {};
#pragma unroll 4
    for (int run = first; run <= last; ++run) {
        const int64_t place = placeOf(run);
        const float2 ml = a.part_ml[place];
        const float f = fastExp2(ml.x - m);
        l += ml.y * f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] += a.part_acc[place * HEAD + 64 * i + lane] * f;
        }
    }
    auto *to = static_cast<typename T::storage *>(a.out) + seq * a.o_stride + head * a.o_head_stride;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        to[64 * i + lane] = T::Base::fromFloat(x[i] * (1.0f / l));
    }
}

} // namespace op::paged_attention_fp4::amd

#endif
