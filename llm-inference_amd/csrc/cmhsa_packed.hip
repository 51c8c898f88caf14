// cmhsa_packed.hip -- causal attention over packed sequences with grouped heads (include/cmhsa_packed.h), MI355X (gfx950).
//
// WORK.  The query heads that share a K/V head become further rows of one problem: sequence s and K/V head g have
// nq * group rows, row r = query r / group, head g * group + r % group.  A workgroup takes 128 of them (four waves of 32)
// through the sequence's keys, 64 (16-bit types) or 32 (fp32) at a time, so a key tile is fetched once for all heads of the
// group and a short sequence with many heads still fills its rows.  Where blocks are few, keys are cut between workgroups, or
// 32 rows are a workgroup and its waves take the keys in turn; sequences of 32 rows and keys take a wave each.
// ARITHMETIC.  S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16: a lane has ONE row (column lane & 31 of S^T and
// O^T), so the softmax needs no traffic between lanes but one exchange of the two lane halves, and what a lane holds of
// S^T after the exponential IS its share of the second product's operand: accumulator register r holds key
// 8 (r / 4) + 4 (lane / 32) + r % 4, and V^T is read with its 16 keys in that order.  V stays as it comes (rows of keys) and
// is transposed by the LDS read itself (ds_read_b64_tr_b16).
// SOFTMAX in the log2 domain, one pass.  Weights are taken against the running maximum of EARLIER tiles; only when a lane's
// sum over the tile leaves [0, 2^12] (2^15 for fp16; always at a row's first tile) is the tile's maximum formed and what was
// accumulated rescaled.  Sums and statistics are fp32; bf16 / fp16 weights are rounded once, to nearest, before the second
// product (half a step of the type: what the output's own rounding costs), and summed as rounded: weights that are off the same
// way are off in numerator and denominator alike (bf16, 32/8 heads of 128, 8192 tokens 571 -> 573 us, 32 heads of 64, 4 x 4096 339 -> 336).
// FP32 runs on the same bf16 matrix instructions: a float is cut into three bf16 parts of 8 bits each, exactly
// (x = hi + mid + lo), and a product is the six part products down to 2^-16 of it; those left out are below 2^-21.  Six
// bf16 instructions take 2.7 times less than the fp32 instruction's time for the same product.
// WHAT IS NOT FINITE.  A masked weight is 0, and 0 times a NaN in V is NaN; an infinity has no three parts.  Whoever
// stages such a value (in a tile that some row does not see all of; for fp32 in any) raises a flag, and the workgroup then
// does its rows over with the plain row loop below, which touches only what a row sees.
// BOUND.  Long sequences: by matrix instructions and the softmax's vector instructions, which the order given in step() lays
// side by side.  Short ones: by a chain of dependent loads (offsets, then keys and queries) and by places for workgroups.
// MEASURED, us (TFLOP/s of the pairs that are seen): bf16, 32/8 heads of 128: 16384 tokens 2218 (991), 4 x 4096 619 (888); 32 heads of
// 64, 4 x 4096 336 (818).  fp32, 16 heads of 64, 8 x 4096 1445 (190), 32/8 of 128, 4096 tokens 760 (181): six times that is
// 1090 of the 1233 that a large bf16 library product reaches.  fp32, 25 heads of 64, 64 prompts of 1..512 tokens 58.8; fp16, 16/4
// heads of 64, 16 x 100 tokens on 4000 61 (423); fp32, 12 heads, 8 tokens 5.1, 300 tokens 11.1.

#include <algorithm>

#include "serving_common.h"

namespace {

using namespace serving;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int kRows = 128;                       // packed rows of a workgroup: four waves of 32

struct PackedParams {
    const void *q, *k, *v;
    void *o;
    int64_t q_rs, k_rs, v_rs, o_rs;
    const int *cu_q, *cu_k;
    int num_seqs, total_q, total_k, num_kv_heads, group, zero_rest;
    float scale_log2;
    float *partial;                              // states of (block, chunk of its keys); null: a block has all its keys to itself
    int *chunk;                                  // behind them: the chunks' length, for the join
    float one_per_target;                        // one over the tickets aimed at for each K/V head
    int min_chunk;                               // the shortest chunk, a multiple of both tile lengths
    int tickets;                                 // of a launch that cuts, for each K/V head
};

// What a workgroup works on: rows first .. first + 128 (or 32) of the (sequence, K/V head) problem of `rows` rows.
struct Block {
    int q0, nq, k0, nk;                          // the sequence's query and key rows
    int first, rows;
    int seq, index;
};

// The offsets of up to 64 sequences, one a lane: everything that follows comes from these registers.
struct Offsets {
    int q0, q1, k0, k1, blocks, each;                            // each: rows of a block, known where this is inlined
    __device__ __forceinline__ explicit Offsets(const PackedParams &p, int rows_each = kRows) : each(rows_each) {
        const int lane = threadIdx.x & 63, at = min(lane, p.num_seqs - 1);
        const int a = p.cu_q[at], b = p.cu_q[at + 1], c = p.cu_k[at], d = p.cu_k[at + 1];
        q0 = clamp_int(a, 0, p.total_q);
        q1 = clamp_int(b, q0, p.total_q);
        k0 = clamp_int(c, 0, p.total_k);
        k1 = clamp_int(d, k0, p.total_k);
        blocks = lane < p.num_seqs ? ((q1 - q0) * p.group + each - 1) / each : 0;
    }
    __device__ __forceinline__ Block block(const PackedParams &p, int s, int index) const {
        Block b;
        b.q0 = __builtin_amdgcn_readlane(q0, s);
        b.nq = __builtin_amdgcn_readlane(q1, s) - b.q0;
        b.k0 = __builtin_amdgcn_readlane(k0, s);
        b.nk = __builtin_amdgcn_readlane(k1, s) - b.k0;
        b.first = index * each;
        b.rows = b.first < b.nq * p.group ? b.nq * p.group : 0;
        b.seq = s;
        b.index = index;
        return b;
    }
    // The t-th block in the order "last blocks of every sequence first": the longest work first.  Found by halving on the
    // block index, with a count over the lanes.
    __device__ __forceinline__ Block block(const PackedParams &p, int t) const {
        if (p.num_seqs == 1) {
            const int n = __builtin_amdgcn_readfirstlane(blocks);
            return block(p, 0, t < n ? n - 1 - t : n);
        }
        if (wave_sum(blocks) <= t) return block(p, 0, 0x7fffff);             // no such block
        int lo = 0, hi = wave_max(blocks);
        while (hi - lo > 1) {                                    // the largest level with more than t blocks at or above it
            const int mid = (lo + hi) >> 1;
            if (wave_sum(max(0, blocks - mid)) > t) lo = mid; else hi = mid;
        }
        const int rank = t - wave_sum(max(0, blocks - lo - 1));
        uint64_t there = __ballot(blocks > lo);                  // the rank-th sequence that has such a block
        for (int i = 0; i < rank; ++i) there &= there - 1;
        return block(p, __builtin_ctzll(there), lo);
    }
};

// Block t where there are more than 64 sequences: sequence s owns the numbers from cu[s] * group / kRows + s on (one more than
// it can need), found by halving.
__device__ __forceinline__ Block block_of_many(const PackedParams &p, int t) {
    Block b;
    int lo = 0, hi = p.num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (clamp_int(p.cu_q[mid], 0, p.total_q) * (int64_t)p.group / kRows + mid <= t) lo = mid; else hi = mid;
    }
    const int s = __builtin_amdgcn_readfirstlane(lo);
    b.q0 = clamp_int(p.cu_q[s], 0, p.total_q);
    b.nq = clamp_int(p.cu_q[s + 1], b.q0, p.total_q) - b.q0;
    b.k0 = clamp_int(p.cu_k[s], 0, p.total_k);
    b.nk = clamp_int(p.cu_k[s + 1], b.k0, p.total_k) - b.k0;
    b.seq = s;
    b.index = max(0, t - (int)(b.q0 * (int64_t)p.group / kRows + s));
    b.first = b.index * kRows;
    b.rows = b.first < b.nq * p.group && t >= (int)(b.q0 * (int64_t)p.group / kRows + s) ? b.nq * p.group : 0;
    return b;
}

// Launches that cut a block's keys (64 sequences at most): a ticket is a block and a chunk of the keys of its sequence.  All
// chunks have one length, so that sum over s of blocks(s) * keys(s), over it, is about the tickets aimed at.  Blocks of
// one chunk lie side by side, so that they find its keys in the cache.
struct Tickets {
    int length, chunks, upto;                                    // the last two: of this lane's sequence
    // (the sum's roundings are less than the 2^-13 added)
    static __device__ __forceinline__ int length_of(const PackedParams &p, const Offsets &o) {
        const float each = fminf(wave_sum((float)o.blocks * (float)(o.k1 - o.k0)) * p.one_per_target * 1.0001f, 1.0e9f);
        return ((int)each + p.min_chunk) / p.min_chunk * p.min_chunk;
    }
    __device__ __forceinline__ Tickets(const Offsets &o, int length) : length(length) {
        chunks = max(1, (o.k1 - o.k0 + length - 1) / length);
        upto = prefix_sum(o.blocks * chunks);
    }
    // the ticket's block and chunk; false if there is none
    __device__ __forceinline__ bool find(const PackedParams &p, const Offsets &o, int t, Block &b, int &chunk) const {
        const int s = __popcll(__ballot(upto <= t));
        if (s >= 64) return false;
        const int rest = t - __builtin_amdgcn_readlane(upto - o.blocks * chunks, s), blocks = __builtin_amdgcn_readlane(o.blocks, s);
        chunk = rest / blocks;
        b = o.block(p, s, rest - chunk * blocks);
        return true;
    }
    // the ticket of a block's first chunk; the next one's is blocks(s) further
    __device__ __forceinline__ int first(const Offsets &o, const Block &b) const { return __builtin_amdgcn_readlane(upto - o.blocks * chunks, b.seq) + b.index; }
};

// floats of a ticket's state: O [kRows][D], m [kRows], l [kRows]
__host__ __device__ constexpr int state_floats(int head_dim) { return kRows * (head_dim + 2); }

// ---------------------------------------------------------------------------------------------------- the plain row loop
// One wave, one packed row: four groups of 16 lanes take the keys j = g, g + 4, .. of [from, to) that the row sees.  The
// result goes to o, or (unfinished) to the row's place in a state.
template <typename T, int D>
__device__ __forceinline__ void plain_row(const PackedParams &p, const Block &b, int kvh, int row, int from, int to, float *state) {
    constexpr int kPer = D / 16;
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int query = row / p.group, head = kvh * p.group + row % p.group;
    const int seen = clamp_int(b.nk - b.nq + query + 1, 0, min(b.nk, to));
    const T *q = static_cast<const T *>(p.q) + (b.q0 + query) * p.q_rs + (int64_t)head * D + c * kPer;
    const T *k = static_cast<const T *>(p.k) + b.k0 * p.k_rs + (int64_t)kvh * D + c * kPer;
    const T *v = static_cast<const T *>(p.v) + b.k0 * p.v_rs + (int64_t)kvh * D + c * kPer;
    T *o = static_cast<T *>(p.o) + (b.q0 + query) * p.o_rs + (int64_t)head * D + c * kPer;
    float qf[kPer], acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { qf[i] = (float)q[i] * p.scale_log2; acc[i] = 0.f; }
    for (int j = from + g; j < seen; j += 4) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) dot += qf[i] * (float)k[j * p.k_rs + i];
        dot = quad_sum(dot);
        dot += dpp_move<0x141>(dot);
        dot += dpp_move<0x140>(dot);
        const float m_new = fmaxf(m, dot);
        const float base = m_new == -INFINITY ? 0.f : m_new;     // seen scores of -inf alone so far: weights 0
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new), e = __builtin_amdgcn_exp2f(dot - base);
        l = l * alpha + e;
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * alpha + e * (float)v[j * p.v_rs + i];
        m = m_new;
    }
    float mt = fmaxf(m, __shfl_xor(m, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mt);      // (weights 0 times what is not finite stay NaN)
    l *= f;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        float a = acc[i] * f;
        a += __shfl_xor(a, 16, 64);
        a += __shfl_xor(a, 32, 64);
        if (g == 0) {
            if (state) state[(row - b.first) * D + c * kPer + i] = a;
            else o[i] = (T)(seen > 0 ? a / l : 0.f);
        }
    }
    if (state && lane == 0) { state[kRows * D + row - b.first] = mt; state[kRows * D + kRows + row - b.first] = l; }
}

// ------------------------------------------------------------------------------------------------------ the tiled kernel
// How a type is computed: its parts, the type of a part, the keys of a tile.
// kLift: weights are taken against 2^-kLift of the maximum; kLimit: the sum over a lane's share of a tile beyond which the
// maximum is formed anew (16 weights of 2^kLift do not pass it).  fp16 has no more than 24 bits below 1: lifted by 8 a weight keeps
// all of its bits down to 2^-22 of the largest and vanishes at 2^-33, so that a long tail below one large weight stays; none
// reaches fp16's 65504.
template <typename T> struct Form { using Part = T; static constexpr int kParts = 1, kKeys = 64; static constexpr float kLift = 0.f, kLimit = 4096.f; };
template <> struct Form<float> { using Part = bf16_t; static constexpr int kParts = 3, kKeys = 32; static constexpr float kLift = 0.f, kLimit = 4096.f; };
template <> struct Form<f16_t> { using Part = f16_t; static constexpr int kParts = 1, kKeys = 64; static constexpr float kLift = 8.f, kLimit = 32768.f; };

__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c, f16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// x = hi + mid + lo, each with 8 bits of x's 24: cutting off, not rounding, so that nothing overflows and nothing is lost
__device__ __forceinline__ void cut(const float (&x)[8], s16x8 (&part)[3]) {
    unsigned h[8], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = __builtin_bit_cast(unsigned, x[i]) & 0xffff0000u;
        const float r = x[i] - __builtin_bit_cast(float, h[i]);
        m[i] = __builtin_bit_cast(unsigned, r) & 0xffff0000u;
        l[i] = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, m[i]));
    }
    u32x4 a, b, c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {                                // the high halves of two words
        a[i] = __builtin_amdgcn_perm(h[2 * i + 1], h[2 * i], 0x07060302);
        b[i] = __builtin_amdgcn_perm(m[2 * i + 1], m[2 * i], 0x07060302);
        c[i] = __builtin_amdgcn_perm(l[2 * i + 1], l[2 * i], 0x07060302);
    }
    part[0] = __builtin_bit_cast(s16x8, a);
    part[1] = __builtin_bit_cast(s16x8, b);
    part[2] = __builtin_bit_cast(s16x8, c);
}

// eight elements as they come from memory
template <typename T> struct Piece { u32x4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(__amdgpu_buffer_rsrc_t from, int offset) {
    Piece<T> x;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = __builtin_amdgcn_raw_buffer_load_b128(from, offset + 16 * i, 0, 0);
    return x;
}
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *from) {
    Piece<T> x;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = reinterpret_cast<const u32x4 *>(from)[i];
    return x;
}
template <typename T> __device__ __forceinline__ void parts_of(const Piece<T> &x, s16x8 (&part)[1]) { part[0] = __builtin_bit_cast(s16x8, x.w[0]); }
__device__ __forceinline__ void parts_of(const Piece<float> &x, s16x8 (&part)[3]) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned w = x.w[i >> 2][i & 3];                   // (a bit cast of the vector's element itself takes element 0)
        f[i] = __builtin_bit_cast(float, w);
    }
    cut(f, part);
}
// whether one of the eight is a NaN or an infinity
template <typename T>
__device__ __forceinline__ bool not_finite(const Piece<T> &x) {
    static_assert(sizeof(T) == 2, "16 bits");
    bool bad = false;
    const unsigned exponent = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned w = x.w[0][j];
        bad |= (w & exponent) == exponent || ((w >> 16) & exponent) == exponent;
    }
    return bad;
}
// bad + 0 x: a NaN from the first of them that is not finite on
__device__ __forceinline__ float times_zero(const Piece<float> &x, float bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned w = x.w[i >> 2][i & 3];
        bad = __builtin_fmaf(__builtin_bit_cast(float, w), 0.f, bad);
    }
    return bad;
}

// weights of eight keys (a lane's registers r .. r + 7) -> the second product's operand
template <typename T, int P>
__device__ __forceinline__ void weights(const float *w, s16x8 (&part)[P]) {
    if constexpr (P == 3) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = w[i];
        cut(f, part);
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (T)w[i];
        part[0] = __builtin_bit_cast(s16x8, x);
    }
}

// sum + the eight elements of a weights' operand, two at a time (off by less than two steps of fp32 a pair)
__device__ __forceinline__ float add_pairs(s16x8 x, float sum, bf16_t) {
    typedef bf16_t t2 __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned pair = w[i];
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(t2, pair), t2{(bf16_t)1.f, (bf16_t)1.f}, sum, false);
    }
    return sum;
}
__device__ __forceinline__ float add_pairs(s16x8 x, float sum, f16_t) {
    typedef f16_t t2 __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned pair = w[i];
        sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(t2, pair), t2{(f16_t)1.f, (f16_t)1.f}, sum, false);
    }
    return sum;
}

// the other lane half's value (lane ^ 32)
__device__ __forceinline__ float other_half(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned y = (threadIdx.x & 32) ? r[0] : r[1];
    return __builtin_bit_cast(float, y);
}

// Rows of no sequence (outside [from, to)) among the 128 rows t * 128 .. of all: zeros, in the columns of a K/V head's group.
template <typename T, int D>
__device__ __forceinline__ void zero_rows(const PackedParams &p, int t, int kvh, int from, int to) {
    if (t * (int64_t)kRows >= from && (t + 1) * (int64_t)kRows <= to) return;
    const int width = p.group * D / 8;
    for (int i = threadIdx.x; i < kRows * width; i += 256) {
        const int64_t row = (int64_t)t * kRows + i / width;
        if (row >= p.total_q) break;
        if (row >= from && row < to) continue;
        float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        store_floats<T, 8>(static_cast<T *>(p.o) + row * p.o_rs + ((int64_t)kvh * width + i % width) * 8, zero);
    }
}

// Which keys a workgroup takes, and which of its tiles every row sees all of.
struct Span { int begin, end, whole, from, to; float *state; };

// A wave's 32 rows: operands, running statistics and sums.
template <typename T, int D>
struct Rows {
    using Part = typename Form<T>::Part;
    static constexpr int P = Form<T>::kParts, KT = Form<T>::kKeys, kPartBytes = KT * D * 2, kSteps = D / 16, kOut = D / 32;
    int query, head, last;                                       // this lane's row, and the last key that it sees
    int k_lane, v_lane;                                          // where the lane reads in a tile of K, of V
    float m, l;                                                  // m: both halves of a row (the maximum less kLift); l: this half's share
    s16x8 q[kSteps][P];
    f32x16 acc[kOut];

    // Returns 0, or a NaN if one of the row's elements is not finite (fp32 only: the others need no parts).
    __device__ __forceinline__ float begin(const PackedParams &p, const Block &b, int kvh, int wave, int lane) {
        const int col = lane & 31, half = lane >> 5;
        const int row = min(b.first + wave * 32 + col, b.rows - 1);      // (the last one again past the end)
        query = row / p.group;
        head = kvh * p.group + row - query * p.group;
        last = b.nk - b.nq + query;
        // Chunk 2 i + half of a key's row lies at 32 i ^ 16 (half ^ (key & 7)) of it, so one exclusive or leads from the first
        // chunk's address to any other's; the same for V.  Tiles and rows are multiples of 128 bytes.
        k_lane = col * D * 2 + 16 * (half ^ (col & 7));
        const int key = 4 * half + ((lane & 15) >> 2);
        v_lane = key * D * 2 + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (2 * (key & 3))) + 8 * (lane & 1);
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
        const T *from = static_cast<const T *>(p.q) + (b.q0 + query) * p.q_rs + (int64_t)head * D + half * 8;
        float bad = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const Piece<T> x = load_piece(from + 16 * i);
            if constexpr (P > 1) bad = times_zero(x, bad);
            parts_of(x, q[i]);
        }
        return bad;
    }

    // c += the product of two operands given in parts, small products first
    static __device__ __forceinline__ void add_products(const s16x8 (&a)[P], const s16x8 (&b)[P], f32x16 &c) {
#pragma unroll
        for (int n = P - 1; n >= 0; --n)
#pragma unroll
            for (int j = 0; j <= n; ++j) c = mfma(a[j], b[n - j], c, Part());
    }

    // S^T of the 32 keys at `k` in LDS
    __device__ __forceinline__ void scores_of(const char *k, f32x16 &next) {
        next = f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            s16x8 y[P];
#pragma unroll
            for (int j = 0; j < P; ++j) y[j] = *reinterpret_cast<const s16x8 *>(k + (k_lane ^ (32 * i)) + j * kPartBytes);
            add_products(y, q[i], next);
        }
    }
    // the scores of 32 keys as weights against `base`: their sum, and the second product's operands.  16-bit weights are summed as
    // they were rounded, so that numerator and denominator have the same error
    __device__ __forceinline__ float weights_of(const f32x16 &s, float scale, float base, s16x8 (&x)[2][P]) {
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float e[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * h + r], scale, -base));
                if constexpr (P > 1) sum += e[r];
            }
            weights<Part, P>(e, x[h]);
            if constexpr (P == 1) sum = add_pairs(x[h][0], sum, Part());
        }
        return sum;
    }
    // One step: the scores of the 32 keys at `k` (the next step's) are formed while those in `s` become weights.  The compiler
    // is told the order: some reads ahead, then a matrix instruction, a read and a share of the vector instructions in turn.
    __device__ __forceinline__ void step(const char *k, f32x16 &next, const f32x16 &s, s16x8 (&x)[2][P], float scale) {
        scores_of(k, next);
        const float sum = weights_of(s, scale, m, x);
        if constexpr (P == 1) {                                  // (fp32 measured better as the compiler orders it)
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (i + 4 < kSteps) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 56 / kSteps, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        settle(s, x, sum, scale);
    }
    // the same without a next step
    __device__ __forceinline__ void weigh(const f32x16 &s, s16x8 (&x)[2][P], float scale) {
        const float sum = weights_of(s, scale, m, x);
        settle(s, x, sum, scale);
    }
    __device__ __forceinline__ void settle(const f32x16 &s, s16x8 (&x)[2][P], float sum, float scale) {
        if (__any(!(sum <= Form<T>::kLimit))) {                  // also a NaN, and a row's first keys (m = -inf): a new maximum
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
            top = fmaxf(top, other_half(top));
            const float m_new = fmaxf(m, top * scale - Form<T>::kLift);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
            for (int i = 0; i < kOut; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
            l *= alpha;
            m = m_new;
            sum = weights_of(s, scale, m_new == -INFINITY ? 0.f : m_new, x);     // nothing seen yet: weights 0
        }
        l += sum;
    }
    // O^T += V^T P^T with the 32 values at `v` in LDS
    __device__ __forceinline__ void accumulate(const char *v, const s16x8 (&x)[2][P]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < kOut; ++i) {
                s16x8 y[P];
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const char *from = v + (v_lane ^ (64 * i)) + j * kPartBytes + h * 32 * D;
                    typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from + 16 * D));         // 8 keys on
                    y[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
                add_products(y, x[h], acc[i]);
            }
    }

    // to o, or unfinished to the block's state
    template <bool kCut>
    __device__ __forceinline__ void finish(const PackedParams &p, const Block &b, float *state, int wave, int lane) {
        const int col = lane & 31, half = lane >> 5, r = wave * 32 + col;
        if (b.first + r >= b.rows) return;
        l += other_half(l);
        if (kCut) {
#pragma unroll
            for (int i = 0; i < kOut; ++i)
#pragma unroll
                for (int j = 0; j < 16; j += 4) *reinterpret_cast<f32x4 *>(state + r * D + 32 * i + 2 * j + 4 * half) = f32x4{acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]};
            if (half == 0) { state[kRows * D + r] = m; state[kRows * D + kRows + r] = l; }
            return;
        }
        const float inv = last < 0 ? 0.f : 1.f / l;
        T *o = static_cast<T *>(p.o) + (b.q0 + query) * p.o_rs + (int64_t)head * D + 4 * half;
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                typedef T t4 __attribute__((ext_vector_type(4)));
                t4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (T)(acc[i][j + e] * inv);
                *reinterpret_cast<t4 *>(o + 32 * i + 2 * j) = x;
            }
    }
};

// The order of a step's second product: the reads of three operands ahead, then a matrix instruction and two reads in turn.
template <int kOut>
__device__ __forceinline__ void sequence_of_products() {
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < 2 * kOut; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (i + 3 < 2 * kOut) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

// scores of 32 keys: those behind `limit` (counted from the lane half's first key) are not seen
__device__ __forceinline__ void hide(f32x16 &s, int limit) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) > limit ? -INFINITY : s[r];
}

// The workgroup's rows once more, one after the other, for what is not finite.
template <typename T, int D>
__device__ __forceinline__ void plain_rows(const PackedParams &p, const Block &b, int kvh, const Span &x, int wave) {
    for (int i = 0; i < 32; ++i) {
        const int r = b.first + wave * 32 + i;
        if (r < b.rows) plain_row<T, D>(p, b, kvh, r, x.from, x.to, x.state);
    }
}

// Sequences of no more than 32 rows and 32 keys, where there are no more than 64: one wave each, four to a workgroup, which
// would otherwise hold its place for one wave's work.  Everything is loaded at once, K as its operands come, V element by
// element (32 lanes 32 consecutive ones), no LDS, no barrier.  64 sequences, 25 heads of 64, us
// so / as blocks: 1 token fp32 8.8 / 23.0, bf16 6.2 / 12.3; 32 tokens 15.1 / 26.4, 9.0 / 14.4.
template <typename T, int D>
__device__ __forceinline__ void short_rows(const PackedParams &p, const Block &b, int kvh, int lane) {
    using R = Rows<T, D>;
    constexpr int P = R::P;
    const int col = lane & 31, half = lane >> 5;
    R rows;
    bool bad = false;
    if (b.nk > 0) {
        const T *k_from = static_cast<const T *>(p.k) + (b.k0 + min(col, b.nk - 1)) * p.k_rs + (int64_t)kvh * D + half * 8;
        const T *v_from = static_cast<const T *>(p.v) + b.k0 * p.v_rs + (int64_t)kvh * D + col;
        Piece<T> k[R::kSteps];
#pragma unroll
        for (int i = 0; i < R::kSteps; ++i) k[i] = load_piece(k_from + 16 * i);
        T v[2][R::kOut][8];                                      // keys in the order of the weights' operand; past the end the last one again
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < R::kOut; ++i) v[h][i][e] = v_from[min(16 * h + 8 * (e >> 2) + 4 * half + (e & 3), b.nk - 1) * p.v_rs + 32 * i];
        float zero = rows.begin(p, b, kvh, 0, lane);
        f32x16 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < R::kSteps; ++i) {
            s16x8 y[P];
            if constexpr (P > 1) zero = times_zero(k[i], zero);
            parts_of(k[i], y);
            R::add_products(y, rows.q[i], s);
        }
        hide(s, rows.last - 4 * half);
        s16x8 weight[2][P];
        rows.weigh(s, weight, p.scale_log2);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < R::kOut; ++i) {
                Piece<T> x;
                __builtin_memcpy(&x, v[h][i], sizeof(x));
                s16x8 y[P];
                if constexpr (P > 1) zero = times_zero(x, zero); else bad |= not_finite(x);
                parts_of(x, y);
                R::add_products(y, weight[h], rows.acc[i]);
            }
        bad |= zero != 0.f;
    } else {
        rows.begin(p, b, kvh, 0, lane);
    }
    if (__any(bad)) plain_rows<T, D>(p, b, kvh, Span{0, 0, 0, 0, 0x7fffffff, nullptr}, 0);
    else rows.template finish<false>(p, b, nullptr, 0, lane);
}

// Block t, or none where the workgroup's waves have done theirs; on the way the rows of no sequence are zeroed.
template <typename T, int D>
__device__ __forceinline__ bool block_or_short_rows(const PackedParams &p, int t, int kvh, Block &b) {
    if (p.num_seqs == 0) {
        if (p.zero_rest) zero_rows<T, D>(p, t, kvh, 0, 0);
        return false;
    }
    if (p.num_seqs > 64) {
        if (p.zero_rest) zero_rows<T, D>(p, t, kvh, p.cu_q[0], p.cu_q[p.num_seqs]);
        b = block_of_many(p, t);
        return true;
    }
    Offsets o(p);
    if (p.zero_rest) zero_rows<T, D>(p, t, kvh, __builtin_amdgcn_readfirstlane(o.q0), __builtin_amdgcn_readlane(o.q1, p.num_seqs - 1));
    const bool is_short = o.blocks == 1 && (o.q1 - o.q0) * p.group <= 32 && o.k1 - o.k0 <= 32;
    if (is_short) o.blocks = 0;
    const int longer = wave_sum(o.blocks);
    if (t < longer) {
        b = o.block(p, t);
        return true;
    }
    uint64_t there = __ballot(is_short);
    const int n = (t - longer) * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (n < __popcll(there)) {
        for (int i = 0; i < n; ++i) there &= there - 1;
        short_rows<T, D>(p, o.block(p, __builtin_ctzll(there), 0), kvh, threadIdx.x & 63);
    }
    return false;
}

// A workgroup's block and keys; false if it has none.
template <typename T, int D, bool kCut, int KT>
__device__ __forceinline__ bool work_of(const PackedParams &p, Block &b, Span &x, int &kvh) {
    kvh = blockIdx.x % p.num_kv_heads;
    const int t = blockIdx.x / p.num_kv_heads;
    x.from = 0;
    x.to = 0x7fffffff;
    x.state = nullptr;
    if (kCut) {
        const Offsets o(p);
        const Tickets y(o, Tickets::length_of(p, o));
        // the join takes it from here: a float sum need not come out alike in two kernels
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.chunk = y.length;
        int chunk;
        if (!y.find(p, o, t, b, chunk)) return false;            // more workgroups than tickets
        x.from = chunk * y.length;
        x.to = x.from + min(y.length, 0x7fffffff - x.from);
        x.state = p.partial + (int64_t)blockIdx.x * state_floats(D);
    } else {
        if (!block_or_short_rows<T, D>(p, t, kvh, b)) return false;
    }
    if (b.rows == 0) return false;
    const int last = b.nk - b.nq + min(b.first + kRows - 1, b.rows - 1) / p.group, first = b.nk - b.nq + b.first / p.group;
    if (kCut && x.from > last) return false;                     // no row sees this chunk
    x.begin = x.from / KT;
    x.end = last >= 0 ? (kCut ? min(last, x.to - 1) : last) / KT + 1 : 0;
    x.whole = first >= 0 ? (first + 1) / KT : 0;
    return true;
}

// Waits until the wave's loads have landed and its LDS reads are done, then for the other waves.
__device__ __forceinline__ void wait_and_meet() {
    __builtin_amdgcn_s_waitcnt(0x0070);                          // vmcnt 0, lgkmcnt 0
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Where a wave's rows of K (or V) come from: `row` and `chunk` (bytes) are the lane's first piece of a tile.
template <typename T, int D, int KT>
struct Source {
    const T *from;
    int row_bytes, keys, row, chunk;
    // asks for the wave's part of the tile that starts at `key`; to: the wave's first place in a buffer.  Rows behind the
    // sequence's last one: that one again
    __device__ __forceinline__ void request(int key, char *to) const {
        constexpr int kChunks = D / 8, kLoads = KT * kChunks / 256;
        const int rows = max(1, min(KT, keys - key));
        key = min(key, keys - 1);
        const auto source = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(from + (int64_t)key * (row_bytes / 2)), 0, (rows - 1) * row_bytes + D * 2, 0x00020000);
#if defined(__HIP_DEVICE_COMPILE__)        // (the host pass checks the 16 against its own target and drops the function)
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(source, (__attribute__((address_space(3))) void *)(to + i * 4096), 16,
                                                     min(row + i * (256 / kChunks), rows - 1) * row_bytes + chunk, 0, 0, 0);
#endif
    }
};

// bf16 and fp16.  Tiles go from memory to LDS without a register between (1 KiB an instruction and wave, the lanes asking for
// the chunks in the order in which they are to lie), two of K and two of V in turn, each under way for the time of a tile;
// a barrier a tile, passed only after the wave's own part has landed.  Scores run half a tile ahead of weights, so tiles of K
// lie half a tile ahead of tiles of V.
template <typename T, int D, bool kCut>
__global__ __launch_bounds__(256, 2) void packed_kernel(PackedParams p) {
    using R = Rows<T, D>;
    constexpr int KT = R::KT, kChunks = D / 8, kLoads = KT * kChunks / 256, kTileBytes = KT * D * 2;
    __shared__ __attribute__((aligned(256))) char lds[4][kTileBytes];        // K, K, V, V
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Block b;
    Span x;
    int kvh;
    if (!work_of<T, D, kCut, KT>(p, b, x, kvh)) return;
    if (tid == 0) flag = 0;

    const T *k_from = static_cast<const T *>(p.k) + b.k0 * p.k_rs + (int64_t)kvh * D;
    const T *v_from = static_cast<const T *>(p.v) + b.k0 * p.v_rs + (int64_t)kvh * D;
    const int k_row = (int)p.k_rs * 2, v_row = (int)p.v_rs * 2;              // bytes; below 2^24
    const int row = tid / kChunks, k_chunk = (tid % kChunks ^ (row & 7)) * 16, v_chunk = (tid % kChunks ^ (2 * (row & 3))) * 16;
    const Source<T, D, KT> ks{k_from, k_row, b.nk, row, k_chunk}, vs{v_from, v_row, b.nk, row, v_chunk};
    R rows;
    bool bad = false;
    if (x.begin < x.end) {
        ks.request(x.begin * KT, &lds[1][wave * 1024]);
        rows.begin(p, b, kvh, wave, lane);
        wait_and_meet();
        ks.request(x.begin * KT + 32, &lds[0][wave * 1024]);
        vs.request(x.begin * KT, &lds[2][wave * 1024]);
        const bool rows_here = b.first + wave * 32 < b.rows;     // a wave without rows helps to fetch only
        const int wave_last = b.nk - b.nq + min(b.first + wave * 32 + 31, b.rows - 1) / p.group;
        f32x16 even, odd;                                        // scores of a tile's first and second 32 keys
        rows.scores_of(lds[1], even);
        for (int tile = x.begin; tile < x.end; ++tile) {
            // V of this tile is there, and the K of its second half and of the next one's first: scores run half a tile ahead
            const int turn = (tile - x.begin) & 1;
            wait_and_meet();
            if (tile + 1 < x.end) {
                ks.request((tile + 1) * KT + 32, &lds[turn ^ 1][wave * 1024]);
                vs.request((tile + 1) * KT, &lds[2 + (turn ^ 1)][wave * 1024]);
            }
            const bool masked = tile >= x.whole;
            if (masked) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    Piece<T> mine;
                    mine.w[0] = *reinterpret_cast<const u32x4 *>(&lds[2 + turn][(i * 256 + tid) * 16]);
                    bad |= not_finite(mine);
                }
            }
            if (rows_here && (!masked || tile * KT <= wave_last)) {
                const int limit = rows.last - tile * KT - 4 * half;
                s16x8 weight[2][1];
                if (masked) hide(even, limit);
                rows.step(lds[turn], odd, even, weight, p.scale_log2);
                rows.accumulate(lds[2 + turn], weight);
                sequence_of_products<R::kOut>();
                if (masked) hide(odd, limit - 32);
                if (masked && tile * KT + 32 > wave_last) continue;          // no row of the wave sees the second half, or what follows
                rows.step(lds[turn] + 64 * D, even, odd, weight, p.scale_log2);
                rows.accumulate(lds[2 + turn] + 64 * D, weight);
                sequence_of_products<R::kOut>();
            }
        }
    } else {
        rows.begin(p, b, kvh, wave, lane);
    }
    if (bad) flag = 1;
    __syncthreads();
    if (flag) plain_rows<T, D>(p, b, kvh, x, wave);              // uniform
    else rows.template finish<kCut>(p, b, x.state, wave, lane);
}

// fp32.  Tiles of 32 keys go through registers, where they are cut into parts: the K of the tile after next and the V of the
// next one are cut between the matrix instructions of this tile's second product, its weights (and their parts) between
// those of the next tile's scores, so that neither pipe waits for the other.  Two tiles of K and two of V in LDS, one
// barrier a tile.
template <int D, bool kCut>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void packed_f32_kernel(PackedParams p) {
    using T = float;
    using R = Rows<T, D>;
    constexpr int P = R::P, KT = R::KT, kChunks = D / 8, kLoads = KT * kChunks / 256, kPartBytes = R::kPartBytes, kTileBytes = P * kPartBytes;
    static_assert(kLoads * 256 == KT * kChunks && KT == 32, "whole pieces, one step a tile");
    // Whether the last tile forms scores of one beyond it (of zeros, used by none) as the others do.  At D = 128 the branch costs the
    // overlap: 4096 tokens, 32/8 heads, 844 us instead of 775; at D = 64 it does not, and a last tile is
    // a large part of a short sequence's work.
    constexpr bool kBeyond = D == 128;
    __shared__ __attribute__((aligned(256))) char lds[4][kTileBytes];        // K, K, V, V, each in parts
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Block b;
    Span x;
    int kvh;
    if (!work_of<T, D, kCut, KT>(p, b, x, kvh)) return;
    if (tid == 0) flag = 0;

    const T *k_from = static_cast<const T *>(p.k) + b.k0 * p.k_rs + (int64_t)kvh * D;
    const T *v_from = static_cast<const T *>(p.v) + b.k0 * p.v_rs + (int64_t)kvh * D;
    const int k_row = (int)p.k_rs * 4, v_row = (int)p.v_rs * 4;
    const int k_at = tid / kChunks * k_row + tid % kChunks * 32, v_at = tid / kChunks * v_row + tid % kChunks * 32;
    // a tile's rows, through a descriptor that ends with the sequence's last row: what lies behind, and tiles that are not
    // this workgroup's, read as zeros
    auto fetch = [&](const T *from, int row_bytes, int at, int tile, Piece<T> (&y)[kLoads]) {
        const int rows = tile < x.end ? min(KT, b.nk - tile * KT) : 0;
        const auto source = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(from + (int64_t)(rows > 0 ? tile : 0) * KT * (row_bytes / 4)), 0,
                                                              rows > 0 ? (rows - 1) * row_bytes + D * 4 : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) y[i] = load_piece<T>(source, at + i * (256 / kChunks) * row_bytes);
    };
    Piece<T> kx[kLoads], vx[kLoads];
    float bad = 0.f;                                             // a NaN once something was not finite
    // Into LDS: pieces of K at chunk ^ (key & 7), of V at chunk ^ 2 (key & 3): the 8 rows that a 128-bit read of K touches
    // at once, and the 4 rows of a transposing read of V, then lie in different banks.
    auto stage = [&](const Piece<T> (&y)[kLoads], char *to, bool values) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int id = tid + 256 * i, r = id / kChunks, c = id % kChunks;
            s16x8 part[P];
            bad = times_zero(y[i], bad);
            parts_of(y[i], part);
#pragma unroll
            for (int j = 0; j < P; ++j) *reinterpret_cast<s16x8 *>(to + j * kPartBytes + (r * kChunks + (c ^ (values ? 2 * (r & 3) : r & 7))) * 16) = part[j];
        }
    };
    R rows;
    if (x.begin < x.end) {
        fetch(k_from, k_row, k_at, x.begin, kx);
        fetch(v_from, v_row, v_at, x.begin, vx);
        bad = rows.begin(p, b, kvh, wave, lane);
        stage(kx, lds[0], false);
        stage(vx, lds[2], true);
        fetch(k_from, k_row, k_at, x.begin + 1, kx);
        __syncthreads();
        f32x16 s, next;
        rows.scores_of(lds[0], s);
        if (x.begin + 1 < x.end) {
            stage(kx, lds[1], false);
            fetch(k_from, k_row, k_at, x.begin + 2, kx);
            fetch(v_from, v_row, v_at, x.begin + 1, vx);
        }
        const bool rows_here = b.first + wave * 32 < b.rows;     // a wave without rows helps to stage only
        const int wave_last = b.nk - b.nq + min(b.first + wave * 32 + 31, b.rows - 1) / p.group;
        for (int tile = x.begin; tile < x.end; ++tile) {
            // in LDS: K of the next tile, V of this one; the scores of this one are formed
            const int turn = (tile - x.begin) & 1;
            const bool masked = tile >= x.whole;
            __syncthreads();
            if (rows_here && (!masked || tile * KT <= wave_last)) {
                s16x8 weight[2][P];
                if (masked) hide(s, rows.last - tile * KT - 4 * half);
                if (kBeyond || tile + 1 < x.end) {
                    rows.step(lds[turn ^ 1], next, s, weight, p.scale_log2);
                    rows.accumulate(lds[2 + turn], weight);
                    stage(kx, lds[turn], false);
                    stage(vx, lds[2 + (turn ^ 1)], true);
                    s = next;
                } else {
                    rows.weigh(s, weight, p.scale_log2);
                    rows.accumulate(lds[2 + turn], weight);
                }
            } else {
                stage(kx, lds[turn], false);
                stage(vx, lds[2 + (turn ^ 1)], true);
            }
            if (kBeyond || tile + 2 < x.end) {
                fetch(k_from, k_row, k_at, tile + 3, kx);
                fetch(v_from, v_row, v_at, tile + 2, vx);
            }
        }
    } else {
        rows.begin(p, b, kvh, wave, lane);
    }
    if (bad != 0.f) flag = 1;
    __syncthreads();
    if (flag) plain_rows<T, D>(p, b, kvh, x, wave);              // uniform
    else rows.template finish<kCut>(p, b, x.state, wave, lane);
}

// Few blocks: 32 rows a workgroup, whose four waves take the 32-key tiles in turn and meet in LDS.  A row's keys then cost a quarter of
// the steps and nothing waits for a barrier on the way, but no two waves share what they load and cut into parts, so this is
// for launches that would leave most of the chip idle.  As in short_rows, K is loaded as its operands come and V element by
// element; a tile is asked for as soon as the registers of the one before are free.
// fp32, 12 heads of 64, 300 tokens 11.1 us, 1024 24.6; bf16, 512 tokens 8.0.
template <typename T, int D>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void packed_waves_kernel(PackedParams p) {
    using R = Rows<T, D>;
    constexpr int P = R::P, kSize = sizeof(T), kPitch = D + 4;   // (the pitch puts the rows of a 16-byte write into different banks)
    __shared__ __attribute__((aligned(16))) float s_o[4][32][kPitch];
    __shared__ float s_m[4][32], s_l[4][32];
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % p.num_kv_heads, t = blockIdx.x / p.num_kv_heads;
    const Offsets o(p, 32);
    if (p.zero_rest) zero_rows<T, D>(p, t, kvh, __builtin_amdgcn_readfirstlane(o.q0), __builtin_amdgcn_readlane(o.q1, p.num_seqs - 1));
    const Block b = o.block(p, t);
    if (b.rows == 0) return;
    if (tid == 0) flag = 0;
    const int last = b.nk - b.nq + min(b.first + 31, b.rows - 1) / p.group, first = b.nk - b.nq + b.first / p.group;
    const int tiles = last >= 0 ? last / 32 + 1 : 0;

    const T *k_from = static_cast<const T *>(p.k) + b.k0 * p.k_rs + (int64_t)kvh * D;
    const T *v_from = static_cast<const T *>(p.v) + b.k0 * p.v_rs + (int64_t)kvh * D;
    const int k_row = (int)p.k_rs * kSize, v_row = (int)p.v_rs * kSize;
    // a tile's rows, through a descriptor that ends with the sequence's last row: what lies behind reads as zeros
    auto source = [&](const T *from, int row_bytes, int tile) {
        const int rows = tile < tiles ? min(32, b.nk - tile * 32) : 0;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(from + (int64_t)(rows > 0 ? tile : 0) * 32 * (row_bytes / kSize)), 0, rows > 0 ? (rows - 1) * row_bytes + D * kSize : 0, 0x00020000);
    };
    Piece<T> k[R::kSteps];
    T v[2][R::kOut][8];                                          // keys in the order of the weights' operand
    auto load_k = [&](int tile) {
        const auto from = source(k_from, k_row, tile);
#pragma unroll
        for (int i = 0; i < R::kSteps; ++i) k[i] = load_piece<T>(from, col * k_row + (half * 8 + 16 * i) * kSize);
    };
    auto load_v = [&](int tile) {
        const auto from = source(v_from, v_row, tile);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < R::kOut; ++i) {
                    const int at = (16 * h + 8 * (e >> 2) + (e & 3) + 4 * half) * v_row + (col + 32 * i) * kSize;
                    if constexpr (kSize == 4) v[h][i][e] = __builtin_bit_cast(T, (unsigned)__builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
                    else v[h][i][e] = __builtin_bit_cast(T, (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0));
                }
    };
    load_k(wave);
    load_v(wave);
    R rows;
    bool bad = false;
    float zero = rows.begin(p, b, kvh, 0, lane);
    for (int tile = wave; tile < tiles; tile += 4) {
        f32x16 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < R::kSteps; ++i) {
            s16x8 y[P];
            if constexpr (P > 1) zero = times_zero(k[i], zero);
            parts_of(k[i], y);
            R::add_products(y, rows.q[i], s);
        }
        load_k(tile + 4);
        const bool masked = tile * 32 + 31 > first;
        if (masked) hide(s, rows.last - tile * 32 - 4 * half);
        s16x8 weight[2][P];
        rows.weigh(s, weight, p.scale_log2);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < R::kOut; ++i) {
                Piece<T> x;
                __builtin_memcpy(&x, v[h][i], sizeof(x));
                s16x8 y[P];
                if constexpr (P > 1) zero = times_zero(x, zero);
                else if (masked) bad |= not_finite(x);
                parts_of(x, y);
                R::add_products(y, weight[h], rows.acc[i]);
            }
        load_v(tile + 4);
    }
    __syncthreads();                                             // flag is 0
    if (bad || zero != 0.f) flag = 1;
    rows.l += other_half(rows.l);
#pragma unroll
    for (int i = 0; i < R::kOut; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) *reinterpret_cast<f32x4 *>(&s_o[wave][col][32 * i + 2 * j + 4 * half]) = f32x4{rows.acc[i][j], rows.acc[i][j + 1], rows.acc[i][j + 2], rows.acc[i][j + 3]};
    if (half == 0) { s_m[wave][col] = rows.m; s_l[wave][col] = rows.l; }
    __syncthreads();
    if (flag) {                                                  // uniform
        for (int i = 0; i < 8; ++i) {
            const int row = b.first + wave * 8 + i;
            if (row < b.rows) plain_row<T, D>(p, b, kvh, row, 0, 0x7fffffff, nullptr);
        }
        return;
    }
    for (int i = tid; i < 8 * D; i += 256) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, row = b.first + r;
        if (row >= b.rows) break;
        const int query = row / p.group, head = kvh * p.group + row - query * p.group;
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = s_m[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][r] - top);
            l += s_l[w][r] * f;
            x += *reinterpret_cast<const f32x4 *>(&s_o[w][r][d]) * f;
        }
        const float inv = b.nk - b.nq + query < 0 ? 0.f : 1.f / l;
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (T)(x[j] * inv);
        *reinterpret_cast<t4 *>(static_cast<T *>(p.o) + (b.q0 + query) * p.o_rs + (int64_t)head * D + d) = y;
    }
}

// Joins the chunks of a block: D / 4 threads a row, 16 (or 32) rows of the 128 a workgroup.
constexpr int kJoinThreads = 512;
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void packed_join_kernel(PackedParams p) {
    constexpr int kThreadsRow = D / 4, kRowsHere = kJoinThreads / kThreadsRow, kParts = kRows / kRowsHere;
    const int part = blockIdx.x % kParts, rest = blockIdx.x / kParts;
    const int kvh = rest % p.num_kv_heads, t = rest / p.num_kv_heads;
    const int length = *p.chunk;                                 // asked for with the offsets, not behind them
    const Offsets places(p);
    if (p.zero_rest && part == 0 && threadIdx.x < 256) zero_rows<T, D>(p, t, kvh, __builtin_amdgcn_readfirstlane(places.q0), __builtin_amdgcn_readlane(places.q1, p.num_seqs - 1));
    const Block b = places.block(p, t);
    if (b.rows == 0) return;
    const Tickets tickets(places, __builtin_amdgcn_readfirstlane(length));
    const int blocks = __builtin_amdgcn_readlane(places.blocks, b.seq), first = tickets.first(places, b);
    const int r = part * kRowsHere + (int)threadIdx.x / kThreadsRow, d = (int)threadIdx.x % kThreadsRow * 4, row = b.first + r;
    if (row >= b.rows) return;
    const int query = row / p.group, head = kvh * p.group + row - query * p.group, last = b.nk - b.nq + query;
    const int count = last >= 0 ? last / tickets.length + 1 : 0;       // chunks that the row sees something of
    if (first < 0 || first + (int64_t)(count - 1) * blocks >= p.tickets) return;     // (offsets that do not ascend: there is no such state)
    const int64_t step = (int64_t)blocks * p.num_kv_heads * state_floats(D);
    const float *state = p.partial + ((int64_t)first * p.num_kv_heads + kvh) * state_floats(D);
    // eight chunks' statistics and sums at once, past the last one its own again with factor 0
    float top = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    constexpr int kAtOnce = 8;
    for (int i = 0; i < count; i += kAtOnce) {
        float m[kAtOnce], part[kAtOnce];
        f32x4 x[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const float *from = state + min(i + j, count - 1) * step;
            m[j] = from[kRows * D + r];
            part[j] = from[kRows * D + kRows + r];
            x[j] = *reinterpret_cast<const f32x4 *>(from + r * D + d);
        }
        float highest = top;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) highest = fmaxf(highest, m[j]);
        const float before = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - highest);
        o *= before;
        l *= before;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const float f = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[j] - highest);
            if (i + j < count) {
                l += part[j] * f;
                o += x[j] * f;
            }
        }
        top = highest;
    }
    const float inv = last < 0 ? 0.f : 1.f / l;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (T)(o[j] * inv);
    *reinterpret_cast<t4 *>(static_cast<T *>(p.o) + (b.q0 + query) * p.o_rs + (int64_t)head * D + d) = y;
}

template <typename T, int D>
void kernels_of(bool cut, bool waves, const void *&fwd, const void *&join) {
    if constexpr (sizeof(T) == 4) fwd = cut ? reinterpret_cast<const void *>(packed_f32_kernel<D, true>) : reinterpret_cast<const void *>(packed_f32_kernel<D, false>);
    else fwd = cut ? reinterpret_cast<const void *>(packed_kernel<T, D, true>) : reinterpret_cast<const void *>(packed_kernel<T, D, false>);
    if (waves) fwd = reinterpret_cast<const void *>(packed_waves_kernel<T, D>);
    join = reinterpret_cast<const void *>(packed_join_kernel<T, D>);
}

// How a launch is laid out.  The host knows the rows, the keys and the sequences, not their lengths.  Measured, in us:
//   waves   32 rows a workgroup, keys in turn to its waves, where such workgroups are few (2 a CU for heads of 64, 4 where they have
//           256 keys or more, 1.5 to 2.5 for heads of 128) and the keys of a sequence, on average, neither fit one tile nor are
//           many.  Not so / so:
//             fp32, 12 heads of 64: 300 tokens 18.3 / 11.1, 1400 38.8 / 34.6, 4 x 512 30.1 / 27.2, 4 x 1 on 1200 18.0 / 22.3 (not), 25 heads,
//             8 x 128 13.3 / 19.6 (not), 8 x 16 on 1000 44 / 21.7; 32/8 heads of 128: 512 tokens 53.7 / 37.6, 1024 101 / 109 (not)
//             bf16, 12 heads of 64: 512 tokens 14.0 / 8.0, 4 x 1 on 2000 14.0 / 19.6 (not), 25 heads, 8 x 16 on 1000 25.4 / 13.4
//             fp16, 12 heads of 64: 2048 tokens 33.5 / 30.1, 4 x 800 22.1 / 24.8 (not), 25 heads, 8 x 1 on 1500 35.2 / 17.1; 16 heads of
//             128, 512 tokens 19.8 / 12.5
//           One sequence may have nearly all the keys: beyond 16384 of them, 128 steps of a wave, a launch that meets the rule for
//           cutting is cut; one that does not is better off here than in blocks, whatever the lengths.  In blocks / cut / so, 16 heads on 4:
//             fp32, 64 x 1 on 1000 48.5 / 43.3 (cut) / 25.0; 25 heads, 15 x 1 on 100 and one on 20000 850 / 94 (cut) / 270
//             bf16, 64 x 1 on 1000 25.7 / 22.2 / 14.4 (so); 25 heads, 15 x 1 on 100 and one on 20000 386 / 40 / 142 (so); 32/8 heads of 128,
//             32 x 1 on 600 23.5 / 30.4 / 17.4 (so)
//   split   otherwise, where all blocks of 128 rows are no more than a round of the chip (4 workgroups a CU for heads of 64, 2 for
//           heads of 128, 1 for fp32 heads of 128) and the sequences' keys are long enough, on average, to pay for the states and
//           the second launch: 1536 (fp32: 768), 768 where half of the CUs would have no workgroup.  Not cut / cut:
//             bf16, 12 heads of 64: 4 x 1 token on 1200 27.0 / 11.6, 4 x 1200 30.4 / 48.0 (not cut)
//             fp32, 12 heads of 64: 4 x 1 token on 800 (cut) 16.2, on 512 25.8, 4 x 512 29.8 / 35.9 (not cut)
//   target  that round (fp16, 16 x 100 tokens on 4000: 64.3, with half of it 67.8; fp32, 2048 tokens: 68 and 92)
struct Plan { bool split, waves; int64_t blocks, tickets; int target; };
Plan plan_of(int num_seqs, int64_t total_q, int64_t total_k, int num_kv_heads, int64_t group, int dtype, int head_dim) {
    Plan plan;
    plan.blocks = total_q * group / kRows + num_seqs;            // no more blocks than that, for each K/V head
    const int64_t waves_blocks = total_q * group / 32 + num_seqs, places = waves_blocks * num_kv_heads, keys = num_seqs > 0 ? total_k / num_seqs : 0;
    const int64_t most = head_dim == 64 ? (keys >= 256 ? 1024 : 512) : dtype == CMHSA_F32 ? 640 : 384;
    const int64_t far = places >= (dtype == CMHSA_F32 ? 256 : 160) ? 2048 : dtype == CMHSA_F32 ? 768 : 1024;
    const bool few = num_seqs > 0 && num_seqs <= 64 && places <= most && keys > 32 && keys <= far;
    const int64_t round = head_dim == 64 ? 1024 : dtype == CMHSA_F32 ? 256 : 512;
    const int64_t least = dtype == CMHSA_F32 || plan.blocks * num_kv_heads <= 128 ? 768 : 1536;
    plan.split = num_seqs > 0 && num_seqs <= 64 && plan.blocks * num_kv_heads <= round && keys >= least && (!few || total_k > 16384);
    plan.waves = few && !plan.split;
    if (plan.waves) plan.blocks = waves_blocks;
    plan.target = (int)std::max<int64_t>(1, round / num_kv_heads);
    plan.tickets = plan.split ? plan.target + plan.blocks + 1 : plan.blocks + 1;
    return plan;
}
size_t states_bytes(const Plan &plan, int num_kv_heads, int head_dim) { return (size_t)plan.tickets * num_kv_heads * state_floats(head_dim) * sizeof(float); }

}  // namespace

extern "C" {

size_t cmhsa_packed_workspace_bytes(int num_seqs, int total_q, int total_k, int num_heads, int num_kv_heads, int head_dim, int dtype) {
    if (num_seqs <= 0 || total_q <= 0 || total_k <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    const Plan plan = plan_of(num_seqs, total_q, total_k, num_kv_heads, num_heads / num_kv_heads, dtype, head_dim);
    return plan.split ? states_bytes(plan, num_kv_heads, head_dim) + 16 : 0;
}

int cmhsa_packed_fwd(const void *q, const void *k, const void *v, void *o,
                     int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride, int64_t o_row_stride,
                     const int *cu_q, const int *cu_k, int num_seqs, int total_q, int total_k,
                     int num_heads, int num_kv_heads, int head_dim, int dtype, int zero_rest,
                     void *workspace, size_t workspace_bytes, void *stream) {
    if (num_seqs < 0 || total_q < 0 || total_k < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads) return CMHSA_ERR_BAD_SHAPE;
    if (dtype != CMHSA_F32 && dtype != CMHSA_BF16 && dtype != CMHSA_F16) return CMHSA_ERR_BAD_SHAPE;
    if (head_dim != 64 && head_dim != 128) return CMHSA_ERR_HEAD_DIM;
    if (total_q == 0 || (num_seqs == 0 && !zero_rest)) return CMHSA_OK;
    if (!q || !o || !cu_q || !cu_k || (total_k && (!k || !v))) return CMHSA_ERR_NULL_POINTER;
    const int64_t size = dtype == CMHSA_F32 ? 4 : 2, d_q = (int64_t)num_heads * head_dim, d_kv = (int64_t)num_kv_heads * head_dim;
    if (q_row_stride < 0 || k_row_stride < 0 || v_row_stride < 0 || o_row_stride < 0) return CMHSA_ERR_BAD_SHAPE;
    if (total_q > 1 && (q_row_stride < d_q || o_row_stride < d_q)) return CMHSA_ERR_BAD_SHAPE;
    if (total_k > 1 && (k_row_stride < d_kv || v_row_stride < d_kv)) return CMHSA_ERR_BAD_SHAPE;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)workspace) & 15) return CMHSA_ERR_ALIGNMENT;
    if (((q_row_stride | k_row_stride | v_row_stride | o_row_stride) * size) & 15) return CMHSA_ERR_ALIGNMENT;
    if (((uintptr_t)cu_q | (uintptr_t)cu_k) & 3) return CMHSA_ERR_ALIGNMENT;
    const int64_t most = (int64_t)1 << 24;                       // bytes of a row
    if (q_row_stride * size >= most || k_row_stride * size >= most || v_row_stride * size >= most || o_row_stride * size >= most) return CMHSA_ERR_TOO_LARGE;
    const int64_t group = num_heads / num_kv_heads;
    if (num_heads > 65535 || total_q * group > 0x7fffffff - 1024 || total_k > 0x7fffffff - 1024) return CMHSA_ERR_TOO_LARGE;
    Plan plan = plan_of(num_seqs, total_q, total_k, num_kv_heads, group, dtype, head_dim);
    if (plan.split && (!workspace || workspace_bytes < cmhsa_packed_workspace_bytes(num_seqs, total_q, total_k, num_heads, num_kv_heads, head_dim, dtype))) {
        plan.split = false;
        plan.tickets = plan.blocks + 1;
    }
    const int parts = kRows * head_dim / 4 / kJoinThreads;               // workgroups of a block in the join
    if (!fits_a_launch(plan.tickets * num_kv_heads, 256)) return CMHSA_ERR_TOO_LARGE;
    if (plan.split && !fits_a_launch((plan.blocks + 1) * num_kv_heads * parts, kJoinThreads)) return CMHSA_ERR_TOO_LARGE;
    PackedParams p;
    p.q = q; p.k = k; p.v = v; p.o = o;
    p.q_rs = q_row_stride; p.k_rs = k_row_stride; p.v_rs = v_row_stride; p.o_rs = o_row_stride;
    p.cu_q = cu_q; p.cu_k = cu_k; p.num_seqs = num_seqs; p.total_q = total_q; p.total_k = total_k;
    p.num_kv_heads = num_kv_heads; p.group = (int)group; p.zero_rest = zero_rest;
    p.scale_log2 = head_dim == 64 ? 0.18033688011112042f : 0.12751743082459868f;      // log2(e) / sqrt(head_dim)
    p.partial = plan.split ? static_cast<float *>(workspace) : nullptr;
    p.chunk = plan.split ? reinterpret_cast<int *>(static_cast<char *>(workspace) + states_bytes(plan, num_kv_heads, head_dim)) : nullptr;
    p.one_per_target = 1.f / (float)plan.target;
    p.min_chunk = 128;                                           // (fp32, 4 x 16 tokens on 1000: 17.1 us, with 256 20.0)
    p.tickets = (int)plan.tickets;
    const void *fwd, *join;
    if (dtype == CMHSA_F32) head_dim == 64 ? kernels_of<float, 64>(plan.split, plan.waves, fwd, join) : kernels_of<float, 128>(plan.split, plan.waves, fwd, join);
    else if (dtype == CMHSA_BF16) head_dim == 64 ? kernels_of<bf16_t, 64>(plan.split, plan.waves, fwd, join) : kernels_of<bf16_t, 128>(plan.split, plan.waves, fwd, join);
    else head_dim == 64 ? kernels_of<f16_t, 64>(plan.split, plan.waves, fwd, join) : kernels_of<f16_t, 128>(plan.split, plan.waves, fwd, join);
    void *args[] = {&p};
    hipError_t e = hipLaunchKernel(fwd, dim3((unsigned)(plan.tickets * num_kv_heads)), dim3(256), args, 0, static_cast<hipStream_t>(stream));
    if (e == hipSuccess && plan.split)
        e = hipLaunchKernel(join, dim3((unsigned)((plan.blocks + 1) * num_kv_heads * parts)), dim3(kJoinThreads), args, 0, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? CMHSA_OK : (int)e;
}

}  // extern "C"
