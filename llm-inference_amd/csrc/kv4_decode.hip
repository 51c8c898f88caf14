// kv4_decode.hip -- one query token a sequence over the paged 4-bit cache (include/cmhsa_kv4.h), MI355X (gfx950).
//
// What has to be read is head_dim * 17 / 16 bytes a key and K/V head; at the card's copy rate a CU gets 7.7 bytes a clock,
// so a key of 128 may cost 17 wave instructions, for all query heads of the group together.  Elementwise products take
// more than that from four query heads on; matrix instructions do not, whatever the group up to 16, and are no slower
// for one.
// ARITHMETIC.  S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_bf16, 32 keys a step and wave.  A code times its
// power of two is exact in bf16, and v_cvt_scalef32_pk_bf16_fp4 makes two of them.  Queries and weights are cut into bf16
// parts instead: fp32 three (exactly), fp16 two (a query exactly, a weight to 2^-16), bf16 one for a query, two for a weight
// (with one, half a step of the output's type, outputs were off by 1.35 times their own rounding; the second costs 1 to 6 %).
// K goes from memory to the operand's registers as it lies: a lane has D / 4 consecutive elements of one key, and the query is
// read in the same order of elements.  V is turned round by LDS: rows of keys in, ds_read_b64_tr_b16 out, the keys in the order
// in which S^T leaves the weights in the registers (so the weights never move).  The wave that writes a V tile reads it: no
// barrier in the loop.  Keys and values of the next step are asked for in the middle of this one, as soon as its registers are
// free.
// SOFTMAX as in cmhsa_packed.hip: weights against the running maximum of earlier steps, a rescale only where a sum leaves
// [0, 2^12]; fp32 statistics; a group of lanes keeps its own sum until the end.
// SPLIT.  Waves of a workgroup take the steps of its keys in turn and meet in LDS.  A long cache is cut into chunks of one
// length for all sequences, chosen from the sum of the lengths (which only the device knows) so that the chunks about
// fill the chip; their states go to the workspace and a second launch joins them.
// MEASURED, us (TB/s of what has to be read): bf16, 32/8 heads of 128, 32 x 16000 keys 108.1 (5.2), 2 x 131000 63.3 (4.5; fp16 64.8,
// fp32 68.3); 25 heads of 64, 64 x 1024, bf16 25.9 (4.3), fp32 31.0 (3.6), 64 of 1 to 1024, fp32 14 to 15: the longest one's steps, and
// 5.9 for 64 of one key; 12 heads, one of 300: 6.0.  A large copy reaches 4.7 TB/s.

#include "kv4_format.h"

namespace {

using namespace serving;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kCols = 16;                        // query heads of one workgroup: the columns of a tile
constexpr float kSumLimit = 4096.f;

struct DecodeParams {
    const void *q;
    void *o;
    int64_t q_rs, o_rs;
    Kv4Pool pool;
    const int *lengths;
    float *partial;                              // states of chunks (null: every sequence is one chunk)
    int2 *heads_of;                              // behind them, for every sequence with keys: (first ticket, chunk length)
    int num_seqs, num_kv_heads, group, head_chunks, num_heads;
    float one_per_head;                          // one over the chunks aimed at, for each K/V head and its head chunk
    int min_chunk, wave_keys;                    // the shortest chunk; the keys a wave takes before another one is used
    float scale_log2;
};

// A length outside [0, capacity] counts as 0.
__device__ __forceinline__ int length_of(const DecodeParams &p, int s) {
    const int n = p.lengths[s];
    return n < 0 || n > ((int64_t)p.pool.table_width << p.pool.page_shift) || p.pool.num_pages == 0 ? 0 : n;
}

// The chunk length of a launch: the sum of the lengths over the chunks aimed at, rounded up, a multiple of 128.  Halves of
// the lengths are added apart (65536 sequences at most: 32 bits hold the sums).
__device__ __forceinline__ int chunk_of(const DecodeParams &p) {
    const int lane = threadIdx.x & 63;
    int low = 0, high = 0;
    for (int at = 0; at < p.num_seqs; at += 64) {
        const int n = at + lane < p.num_seqs ? length_of(p, at + lane) : 0;
        low += n & 0xffff;
        high += n >> 16;
    }
    low = __builtin_amdgcn_readlane(prefix_sum(low), 63);
    high = __builtin_amdgcn_readlane(prefix_sum(high), 63);
    // A little above total / per_head whatever the roundings (each below 2^-23 of it), so that no more than
    // per_head + num_seqs chunks come out; no sequence is longer than 2^31 - 1025.
    const float each = ((float)high * 65536.f + (float)(unsigned)low) * p.one_per_head * 1.000001f;
    return max(p.min_chunk, ((int)fminf(each, 2147483000.f - 512.f) + 128) / 128 * 128);
}

__device__ __forceinline__ int chunks_of(int n, int chunk) { return (int)(((unsigned)n + (unsigned)chunk - 1) / (unsigned)chunk); }       // (the sum may pass 2^31)

// eight codes of one scale -> a matrix operand
__device__ __forceinline__ s16x8 operand(unsigned codes, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    const u32x4 x = {__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, c), __builtin_bit_cast(unsigned, d)};
    return __builtin_bit_cast(s16x8, x);
}

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// eight floats -> P bf16 parts that add up to them (P = 1: rounded to nearest)
template <int P>
__device__ __forceinline__ void parts_of(const float (&x)[8], s16x8 (&part)[P]) {
    if constexpr (P == 1) {
        bf16x8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (bf16_t)x[i];
        part[0] = __builtin_bit_cast(s16x8, y);
    } else {
        unsigned rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = __builtin_bit_cast(unsigned, x[i]);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(rest[2 * i + 1], rest[2 * i], 0x07060302);      // the high halves of two words
            part[j] = __builtin_bit_cast(s16x8, w);
            if (j + 1 < P)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r = __builtin_bit_cast(float, rest[i]) - __builtin_bit_cast(float, rest[i] & 0xffff0000u);
                    rest[i] = __builtin_bit_cast(unsigned, r);
                }
        }
    }
}

template <typename T> struct Parts { static constexpr int n = 1; };
template <> struct Parts<f16_t> { static constexpr int n = 2; };
template <> struct Parts<float> { static constexpr int n = 3; };

// the maximum over the four lanes that have the same column (lane, lane ^ 16, lane ^ 32, lane ^ 48)
__device__ __forceinline__ float column_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float column_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// floats of one chunk's state: O [heads][D], m [heads], l [heads]
__host__ __device__ constexpr int state_floats(int heads, int head_dim) { return heads * (head_dim + 2); }

// What a wave requests for a step: two subtiles of 16 keys, each within one page.  (64 keys a step for heads of 64 would
// have half the steps, and measured slower: 64 sequences of up to 1024, 18.9 us against 15.8.)
template <int D>
struct Keys {
    static constexpr int kSub = 2, kWords = D / 32;              // words of codes: a lane has D / 4 elements of a key
    typedef unsigned words __attribute__((ext_vector_type(kWords)));
    words k[kSub], v[kSub];
    unsigned ks[kSub], vs[kSub];
    int first[kSub];                                             // position of a subtile's first key; past the end where there is no page
};

template <typename T, int D, int W>
__global__ __launch_bounds__(W * 64, D == 128 && Parts<T>::n > 1 ? 3 : 4) void decode_kernel(DecodeParams p) {
    constexpr int P = Parts<T>::n, kWeightParts = P == 1 ? 2 : P, kWords = D / 32, kTiles = D / 16, kChunks = D / 8;
    constexpr int kSub = Keys<D>::kSub, kStep = 16 * kSub;
    constexpr int kWaveBytes = kStep * D * 2;                    // a wave's V tile; its O state goes there at the end
    static_assert(kWaveBytes >= kCols * D * 4, "one area for both");
    __shared__ __attribute__((aligned(16))) char lds[W][kWaveBytes];
    __shared__ float s_m[W][kCols], s_l[W][kCols];

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per_ticket = p.num_kv_heads * p.head_chunks;
    const int ticket = blockIdx.x / per_ticket, rest = blockIdx.x - ticket * per_ticket;
    const int kvh = rest / p.head_chunks, h0 = (rest - kvh * p.head_chunks) * kCols, heads = min(kCols, p.group - h0);

    // the ticket's sequence and keys, and the query: column h0 + col, elements in the order of K's lanes
    float qf[kWords][8];
    auto load_query = [&](int seq) {
        const T *src = static_cast<const T *>(p.q) + seq * p.q_rs + (int64_t)(kvh * p.group + h0 + min(col, heads - 1)) * D + quarter * (D / 4);
#pragma unroll
        for (int i = 0; i < kWords; ++i) load_floats<T, 8>(src + 8 * i, qf[i]);
    };
    int s, from, to;
    if (p.partial) {
        const int chunk = chunk_of(p);
        int before = 0;
        s = -1;
        for (int at = 0; at < p.num_seqs; at += 64) {
            const int n = at + lane < p.num_seqs ? length_of(p, at + lane) : 0;
            const int count = chunks_of(n, chunk);
            const int upto = prefix_sum(count);
            const int here = __popcll(__ballot(before + upto <= ticket));      // sequences that end before the ticket
            if (here < 64) {
                s = at + here;
                from = (ticket - before - __builtin_amdgcn_readlane(upto - count, here)) * chunk;
                to = from + min(chunk, __builtin_amdgcn_readlane(n, here) - from);
                break;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        if (s < 0 || s >= p.num_seqs) return;                    // more workgroups than chunks
        if (from == 0 && rest == 0 && tid == 0) p.heads_of[s] = int2{ticket, chunk};      // for the join: the sequence's first ticket
    } else {
        s = ticket;
        from = to = 0;
    }

    const int size = 1 << p.pool.page_shift;
    const int *table = p.pool.table + s * p.pool.table_stride;
    // Waves without keys leave at once (a barrier waits for those that are left only): in a batch of short sequences they
    // would hold the places of other workgroups' waves.  The first wave does not wait for the length before it asks for the
    // page numbers and the query.
    auto waves_of = [&]() { return max(1, min(W, (to - from + p.wave_keys - 1) / p.wave_keys)); };
    if (!p.partial && wave > 0) to = __builtin_amdgcn_readfirstlane(length_of(p, s));
    if ((p.partial || wave > 0) && wave >= waves_of()) return;
    // The page numbers of 64 consecutive pages lie in a register, one a lane, those of the next 64 in another; a step reads
    // its own with v_readlane.  (Loaded one by one as scalars they would hold up every LDS read behind them: both count
    // on the same counter, and scalar loads return in any order.)
    int base = (from + wave * kStep) >> p.pool.page_shift, mine = -1, ahead = -1;
    if (p.pool.table_width > 0) {
        mine = table[min(base + lane, p.pool.table_width - 1)];
        ahead = table[min(base + 64 + lane, p.pool.table_width - 1)];
    }
    load_query(s);
    if (!p.partial && wave == 0) to = __builtin_amdgcn_readfirstlane(length_of(p, s));
    asm volatile("" ::"v"(mine), "v"(ahead), "s"(to));           // asked for together, not one after the other
    const int waves = waves_of();
    const uint8_t *pool = p.pool.pages + (int64_t)kvh * CMHSA_KV4_BLOCK_BYTES(size, D);
    const int code_at = col * (D / 2) + quarter * (D / 8), scale_byte = col * (D / 32) + quarter * (D / 4) / 32;
    const int scale_at = scale_byte & -4, scale_shift = 8 * (scale_byte & 3);        // scale bytes come as the word around them

    auto pages_of = [&](int at, int (&page)[kSub]) {             // a subtile that starts behind `to` takes the last page
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            const int n = min(at + 16 * u, to - 1) >> p.pool.page_shift;
            if (n - base >= 64) {                                // uniform, and never more than one block of 64 on: a step's reach is less
                base += 64;
                mine = ahead;
                ahead = table[min(base + 64 + lane, p.pool.table_width - 1)];
                asm volatile("" : "+v"(ahead));                  // waited for here, so that the loop's own waits can be exact
            }
            page[u] = __builtin_amdgcn_readlane(mine, n - base);
        }
    };
    auto request = [&](int at, Keys<D> &x) {
        int page[kSub];
        pages_of(at, page);
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            const bool there = (unsigned)page[u] < (unsigned)p.pool.num_pages;
            x.first[u] = there ? at + 16 * u : 0x7fffff00;
            const uint8_t *block = pool + (there ? page[u] : 0) * p.pool.page_stride;
            const int slot = (at + 16 * u) & (size - 1);
            const uint8_t *codes = block + slot * (D / 2), *scales = block + size * D + slot * (D / 32);
            x.k[u] = *reinterpret_cast<const typename Keys<D>::words *>(codes + code_at);
            x.v[u] = *reinterpret_cast<const typename Keys<D>::words *>(codes + size * (D / 2) + code_at);
            x.ks[u] = *reinterpret_cast<const unsigned *>(scales + scale_at);
            x.vs[u] = *reinterpret_cast<const unsigned *>(scales + size * (D / 32) + scale_at);
        }
    };

    f32x4 acc[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool seen = false;                                           // uniform: a key counts, whatever its score

    const int stride = waves * kStep;
    int at = from + wave * kStep;
    if (at < to) {
        Keys<D> x;
        request(at, x);
        s16x8 q[kWords][P];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) qf[i][j] = col < heads ? qf[i][j] : 0.f;         // columns past the group are zeros
            parts_of<P>(qf[i], q[i]);
        }
        char *tile = lds[wave];
        for (; at < to; at += stride) {
            bool masked = false;                                 // uniform: a subtile that ends past `to`, or has no page
#pragma unroll
            for (int u = 0; u < kSub; ++u) { masked |= x.first[u] > to - 16; seen |= x.first[u] < to; }
            // scores: rows of S^T are keys 4 quarter + r of each subtile
            float w[kSub][4];
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const float scale = kv4_scale(x.ks[u] >> scale_shift & 255);
                f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const s16x8 k = operand(x.k[u][i], scale);
#pragma unroll
                    for (int j = P - 1; j >= 0; --j) y = mfma(k, q[i][j], y);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) w[u][r] = y[r];
            }
            // V, as bf16 rows of keys: piece c of key r at c ^ f(r), where f takes all 8 values over 8 keys (a write) and
            // puts 4 keys into the 4 32-byte quarters of 128 bytes (a transposing read)
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const int r = 16 * u + col;
                const unsigned byte = masked && x.first[u] + col >= to ? 0u : x.vs[u] >> scale_shift & 255;      // a key that does not count: finite, whatever lies there
                const float scale = kv4_scale(byte);
#pragma unroll
                for (int i = 0; i < kWords; ++i)
                    *reinterpret_cast<s16x8 *>(tile + (r * kChunks + ((quarter * kWords + i) ^ (2 * (r & 3) + ((r >> 2) & 1)))) * 16) = operand(x.v[u][i], scale);
            }
            int first[kSub];
#pragma unroll
            for (int u = 0; u < kSub; ++u) first[u] = x.first[u];
            // the next step's, into the registers that this one is done with (past the end the last keys again, unused: the
            // number of loads on their way stays known, and waits exact)
            request(min(at + stride, to - 1) & -16, x);
            if (masked)
#pragma unroll
                for (int u = 0; u < kSub; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (first[u] + 4 * quarter + r >= to) w[u][r] = -INFINITY;
            float e[kSub / 2][8], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4 * kSub; ++i) { e[i >> 3][i & 7] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[i >> 2][i & 3], p.scale_log2, -m)); sum += e[i >> 3][i & 7]; }
            if (__any(!(sum <= kSumLimit))) {                    // also a NaN, and a wave's first step (m = -inf)
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4 * kSub; ++i) top = fmaxf(top, w[i >> 2][i & 3]);
                const float m_new = fmaxf(m, column_max(top) * p.scale_log2);
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                const float base = m_new == -INFINITY ? 0.f : m_new;         // no key yet: weights 0
#pragma unroll
                for (int i = 0; i < kTiles; ++i) acc[i] *= alpha;
                l *= alpha;
                m = m_new;
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4 * kSub; ++i) { e[i >> 3][i & 7] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[i >> 2][i & 3], p.scale_log2, -base)); sum += e[i >> 3][i & 7]; }
            }
            l += sum;
            __builtin_amdgcn_wave_barrier();                     // the tile's writes stay in front of its reads (one wave's LDS accesses run in order)
#pragma unroll
            for (int half = 0; half < kSub / 2; ++half) {        // 32 keys
                s16x8 weight[kWeightParts];
                parts_of<kWeightParts>(e[half], weight);
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const int r = 32 * half + 4 * quarter + (col >> 2), c = 2 * i + ((col & 3) >> 1);
                    const char *base = tile + (r * kChunks + (c ^ (2 * (r & 3) + ((r >> 2) & 1)))) * 16 + (col & 1) * 8;
                    typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(base));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(base + 16 * kChunks * 16));   // 16 keys on: the same f
                    const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int j = kWeightParts - 1; j >= 0; --j) acc[i] = mfma(v, weight[j], acc[i]);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    // the waves' states meet in LDS: O [col][D] in the wave's own area.  A wave whose scores are all -inf has the lowest finite maximum: beside
    // others it weighs nothing, and alone the result is 0 / 0; -inf is left for those that have no key.
    l = column_sum(l);
    if (seen && m == -INFINITY) m = -3.4028234663852886e38f;
    __builtin_amdgcn_wave_barrier();
    float *state = reinterpret_cast<float *>(lds[wave]);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) *reinterpret_cast<f32x4 *>(state + col * D + 16 * i + 4 * quarter) = acc[i];
    if (quarter == 0) { s_m[wave][col] = m; s_l[wave][col] = l; }
    if (waves > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
    float *out = p.partial ? p.partial + (int64_t)blockIdx.x * state_floats(kCols, D) : nullptr;
    for (int i = tid; i < heads * D; i += waves * 64) {
        const int h = i / D, d = i % D;
        float mt = -INFINITY, lt = 0.f, ot = 0.f;
        for (int w = 0; w < waves; ++w) mt = fmaxf(mt, s_m[w][h]);
        for (int w = 0; w < waves; ++w) {
            const float f = s_m[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][h] - mt);
            lt += s_l[w][h] * f;
            ot += reinterpret_cast<const float *>(lds[w])[h * D + d] * f;
        }
        if (out) {
            out[h * D + d] = ot;
            if (d == 0) { out[kCols * D + h] = mt; out[kCols * D + kCols + h] = lt; }
        } else {
            static_cast<T *>(p.o)[s * p.o_rs + (int64_t)(kvh * p.group + h0 + h) * D + d] = (T)(mt == -INFINITY && lt == 0.f ? 0.f : ot / lt);
        }
    }
}

// Joins the chunks of a sequence: one workgroup per (sequence, query head), 256 / D chunks at a time.  The weights of 256
// chunks go to LDS first, so that the states themselves are read without waiting for one another.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(DecodeParams p) {
    constexpr int kParts = 256 / D;
    __shared__ float s_top[4], s_sum[4], s_f[256], s_o[kParts][D];
    const int tid = threadIdx.x, lane = tid & 63, d = tid % D, part = tid / D;
    const int s = blockIdx.x / p.num_heads, head = blockIdx.x - s * p.num_heads;
    const int kvh = head / p.group, in_group = head - kvh * p.group, h = in_group % kCols;
    const int per_ticket = p.num_kv_heads * p.head_chunks;
    const int n = length_of(p, s);
    const int2 place = p.heads_of[s];                            // (not written, and not used, where n is 0)
    const int count = n > 0 ? chunks_of(n, place.y) : 0;
    const float *first = p.partial + ((int64_t)(n > 0 ? place.x : 0) * per_ticket + kvh * p.head_chunks + in_group / kCols) * state_floats(kCols, D);
    const int64_t step = (int64_t)per_ticket * state_floats(kCols, D);
    const float *maxima = first + kCols * D + h, *sums = maxima + kCols;
    float top = -INFINITY;
    for (int i = tid; i < count; i += 256) top = fmaxf(top, maxima[i * step]);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    if (lane == 0) s_top[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    float o = 0.f, l = 0.f;
    for (int at = 0; at < count; at += 256) {
        float f = 0.f;
        if (at + tid < count) {
            const float m = maxima[(at + tid) * step];
            f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
            l += sums[(at + tid) * step] * f;
        }
        __syncthreads();                                         // the weights before have been read
        s_f[tid] = f;
        __syncthreads();
        const int n = min(count - at, 256);
        const float *from = first + at * step + h * D + d;
#pragma unroll 8
        for (int i = part; i < n; i += kParts) o += from[i * step] * s_f[i];
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x, 64);
    if (lane == 0) s_sum[tid >> 6] = l;
    s_o[part][d] = o;
    __syncthreads();
    if (tid < D) {
        l = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
#pragma unroll
        for (int i = 1; i < kParts; ++i) o += s_o[i][d];
        static_cast<T *>(p.o)[s * p.o_rs + (int64_t)head * D + d] = (T)(top == -INFINITY && l == 0.f ? 0.f : o / l);
    }
}

template <typename T, int D>
void kernels_of(int waves, const void *&decode, const void *&join) {
    decode = waves == 4 ? reinterpret_cast<const void *>(decode_kernel<T, D, 4>) : reinterpret_cast<const void *>(decode_kernel<T, D, 8>);
    join = reinterpret_cast<const void *>(join_kernel<T, D>);
}

// How a launch is laid out, by sizes that the host knows (the lengths themselves it does not).  Measured, in us a call:
//   split      beyond 1024 positions where the workgroups would be few (12 of 2000 positions: 9.4 cut and joined, 12.4 not;
//              96 of 1200: 10.9 and 9.8), beyond 2048 (1600, one sequence of 4096 among 63 of 500: 28 and 34; all of
//              4096: 115 and 109) unless sequences are so many that every workgroup's look through their lengths costs more
//              than one long sequence alone would: workgroups times sequences against 256 times the capacity.  Not cut / cut,
//              all of 1000 and one as long as the table: 1024 x 8 K/V heads of 128, table of 16384 (512 times) 213 / 318, 303 / 388;
//              of 131072 (64 times) 205 / 322, 1147 / 417; 256 x 8, of 16384 (32) 51 / 69, 158 / 89; 4096 x 1 of 64, of 4096 (4096) 53 / 180, 67 / 184
//   per_head   chunks aimed at: one round of the chip, 3 workgroups a CU for heads of 128 (two of 131000, fp16: 65.4, and
//              73.5 with 4 a CU, of which the last would wait), 4 for heads of 64
//   waves      8 where few workgroups hold a sequence each (256 of 1000: 11.2, and 12.3 with 4), else 4
//   wave_keys  two steps a wave before another wave joins in where waves are many (1600 workgroups of 128 positions: 9.8, and
//              11.6 with one), one step where they are few
struct Plan { int head_chunks, per_head, waves, wave_keys, min_chunk; bool split; int64_t tickets; };
Plan plan_of(int num_seqs, int64_t capacity, int num_heads, int num_kv_heads, int head_dim) {
    Plan plan;
    plan.head_chunks = (num_heads / num_kv_heads + kCols - 1) / kCols;
    const int64_t each = (int64_t)num_kv_heads * plan.head_chunks, all = each * num_seqs, round = head_dim == 128 ? 768 : 1024;
    plan.split = (capacity > 2048 || (capacity > 1024 && all < 64)) && num_seqs <= 65536 && all * num_seqs <= 256 * capacity;
    plan.per_head = (int)(each >= round ? 1 : round / each);
    plan.waves = plan.split || all >= 512 ? 4 : 8;
    plan.wave_keys = all >= 1024 ? 64 : 32;
    plan.min_chunk = 256;
    plan.tickets = plan.split ? (int64_t)plan.per_head + num_seqs : num_seqs;
    return plan;
}
size_t states_bytes(const Plan &plan, int num_kv_heads, int head_dim) {
    return (size_t)plan.tickets * num_kv_heads * plan.head_chunks * state_floats(kCols, head_dim) * sizeof(float);
}

}  // namespace

extern "C" {

size_t cmhsa_kv4_decode_workspace_bytes(int num_seqs, int table_width, int page_size, int num_heads, int num_kv_heads, int head_dim) {
    if (num_seqs <= 0 || table_width <= 0 || page_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    const Plan plan = plan_of(num_seqs, (int64_t)table_width * page_size, num_heads, num_kv_heads, head_dim);
    return plan.split ? states_bytes(plan, num_kv_heads, head_dim) + num_seqs * sizeof(int2) : 0;
}

int cmhsa_kv4_decode(const void *q, void *o, int64_t q_row_stride, int64_t o_row_stride, int dtype,
                     const uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *lengths, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                     void *workspace, size_t workspace_bytes, void *stream) {
    if (num_seqs < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads) return CMHSA_ERR_BAD_SHAPE;
    if (dtype != CMHSA_F32 && dtype != CMHSA_BF16 && dtype != CMHSA_F16) return CMHSA_ERR_BAD_SHAPE;
    const int bad = kv4_check_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width, num_kv_heads, head_dim);
    if (bad) return bad;
    if (num_seqs == 0) return CMHSA_OK;
    if (!q || !o || !lengths) return CMHSA_ERR_NULL_POINTER;
    const int64_t size = dtype == CMHSA_F32 ? 4 : 2, d_q = (int64_t)num_heads * head_dim;
    if (q_row_stride < 0 || o_row_stride < 0 || (num_seqs > 1 && (q_row_stride < d_q || o_row_stride < d_q))) return CMHSA_ERR_BAD_SHAPE;
    if ((((uintptr_t)q | (uintptr_t)o | (uintptr_t)workspace) & 15) || (((q_row_stride | o_row_stride) * size) & 15) || ((uintptr_t)lengths & 3)) return CMHSA_ERR_ALIGNMENT;
    const Plan plan = plan_of(num_seqs, (int64_t)table_width * page_size, num_heads, num_kv_heads, head_dim);
    if (plan.split && (!workspace || workspace_bytes < cmhsa_kv4_decode_workspace_bytes(num_seqs, table_width, page_size, num_heads, num_kv_heads, head_dim)))
        return CMHSA_ERR_WORKSPACE;
    const int64_t grid = plan.tickets * num_kv_heads * plan.head_chunks;
    if (!fits_a_launch(grid, plan.waves * 64) || (plan.split && !fits_a_launch((int64_t)num_seqs * num_heads, 256))) return CMHSA_ERR_TOO_LARGE;
    DecodeParams p;
    p.q = q; p.o = o; p.q_rs = q_row_stride; p.o_rs = o_row_stride;
    p.pool = kv4_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width);
    p.lengths = lengths;
    p.partial = plan.split ? static_cast<float *>(workspace) : nullptr;
    p.heads_of = plan.split ? reinterpret_cast<int2 *>(static_cast<char *>(workspace) + states_bytes(plan, num_kv_heads, head_dim)) : nullptr;
    p.num_seqs = num_seqs; p.num_kv_heads = num_kv_heads; p.group = num_heads / num_kv_heads; p.head_chunks = plan.head_chunks; p.num_heads = num_heads;
    p.one_per_head = 1.f / (float)plan.per_head;
    p.min_chunk = plan.min_chunk;
    p.wave_keys = plan.wave_keys;
    p.scale_log2 = head_dim == 64 ? 0.18033688011112042f : 0.12751743082459868f;      // log2(e) / sqrt(head_dim)
    const void *decode, *join;
    if (dtype == CMHSA_F32) head_dim == 64 ? kernels_of<float, 64>(plan.waves, decode, join) : kernels_of<float, 128>(plan.waves, decode, join);
    else if (dtype == CMHSA_BF16) head_dim == 64 ? kernels_of<bf16_t, 64>(plan.waves, decode, join) : kernels_of<bf16_t, 128>(plan.waves, decode, join);
    else head_dim == 64 ? kernels_of<f16_t, 64>(plan.waves, decode, join) : kernels_of<f16_t, 128>(plan.waves, decode, join);
    void *args[] = {&p};
    hipError_t e = hipLaunchKernel(decode, dim3((unsigned)grid), dim3(plan.waves * 64), args, 0, static_cast<hipStream_t>(stream));
    if (e == hipSuccess && plan.split) e = hipLaunchKernel(join, dim3((unsigned)(num_seqs * num_heads)), dim3(256), args, 0, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? CMHSA_OK : (int)e;
}

}  // extern "C"
