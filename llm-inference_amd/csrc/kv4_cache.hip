// kv4_cache.hip -- storing into the paged 4-bit cache, reading it back, copying its pages (include/cmhsa_kv4.h), MI355X.
//
// All three are copies with a conversion on the way: bound by HBM where they are large, by the launch where they are one
// token a sequence.
//   append / gather: a wave takes 512 elements of K or V of one row or of four; a lane has 8 consecutive elements (16 or 32 bytes
//     of values, 4 bytes of codes), a quad of lanes one block of 32.  A row's sequence: one load of the offsets and a ballot.
//     append's loads of values go out before that search.  48019 rows of 8 heads of 128, bf16, in 12 prompts: append 53.7 us,
//     gather 51.9, 4.6 and 4.8 TB/s of what has to be read and written, the rate of a large copy.  64 rows of 25 heads of 64, fp32:
//     3.0 us in a graph, a chain of four dependent loads.
//   copy: a grid of (16-KiB piece, pair, layer); the pairs ride in the kernel's arguments, so that nothing is uploaded.

#include "kv4_format.h"

namespace {

using namespace serving;

struct RowsParams {
    const void *k_in, *v_in;
    void *k_out, *v_out;
    int64_t k_rs, v_rs;
    Kv4Pool pool;
    const int *cu, *starts;
    int num_seqs, rows, width, chunks, zero_rest;      // width = num_kv_heads * head_dim, chunks = ceil(width / 512)
};

// A wave's place in the work: K or V, its first row, the lane's first element; and of each row r, in lane r, the page (-1: it has
// none) and the slot.  `owned` has a bit for each row that belongs to a sequence.
template <int R>
struct Places {
    int which, row, element, page, slot;
    unsigned owned;

    __device__ __forceinline__ explicit Places(const RowsParams &p) {
        const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (int)(threadIdx.x >> 6));
        const int group = id / (2 * p.chunks), rest = id - group * 2 * p.chunks;
        which = rest >= p.chunks;
        row = group * R;
        element = (rest - which * p.chunks) * 512 + (int)(threadIdx.x & 63) * 8;
    }
    // one load of up to 64 sequences' offsets and starts, a count of the ends at or before each row, one load of the pages
    __device__ __forceinline__ void find(const RowsParams &p) {
        const int lane = threadIdx.x & 63;
        int first = 0, end = 0x7fffffff, start = 0, lo = 0;
        auto look = [&] {
            const int s = lo + lane;
            if (s < p.num_seqs) {
                first = p.cu[s];
                end = p.cu[s + 1];
                if (p.starts) start = p.starts[s];
            } else {
                end = 0x7fffffff;
            }
        };
        if (p.num_seqs <= 64) look();
        int seq = 0;
        int64_t position = -1;
        owned = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (p.num_seqs > 64) {                               // the answer lies in [lo, hi]: halved down to a wave of candidates
                lo = 0;
                int hi = p.num_seqs;
                while (hi - lo > 63) {
                    const int mid = (lo + hi) >> 1;
                    if (p.cu[mid + 1] <= row + r) lo = mid + 1; else hi = mid;
                }
                look();
            }
            const int at = __popcll(__ballot(end <= row + r)), s = lo + at;
            if (s >= p.num_seqs || row + r >= p.rows) continue;  // uniform: behind the last sequence
            const int from = __builtin_amdgcn_readlane(first, at), begin = __builtin_amdgcn_readlane(start, at);
            if (row + r < from) continue;
            owned |= 1u << r;
            if (lane == r) {
                seq = s;
                position = (int64_t)begin + (row + r - (int64_t)from);
            }
        }
        page = -1;
        slot = (int)position & ((1 << p.pool.page_shift) - 1);
        if (position >= 0 && position < ((int64_t)p.pool.table_width << p.pool.page_shift)) page = kv4_page(p.pool, seq, (int)position);
    }
    // row r's codes and scale byte of the lane's 8 elements
    template <int D>
    __device__ __forceinline__ void addresses(const RowsParams &p, int r, uint8_t *&codes, uint8_t *&scale) const {
        const int size = 1 << p.pool.page_shift, head = element / D, d = element % D;
        const int at = which * size + __builtin_amdgcn_readlane(slot, r);
        uint8_t *block = p.pool.pages + __builtin_amdgcn_readlane(page, r) * p.pool.page_stride + (int64_t)head * CMHSA_KV4_BLOCK_BYTES(size, D);
        codes = block + at * (D / 2) + d / 2;
        scale = block + size * D + at * (D / 32) + d / 32;
    }
};

template <typename T, int D, int R>
__global__ __launch_bounds__(256) void append_kernel(RowsParams p) {
    Places<R> w(p);
    if (w.row >= p.rows) return;                                 // wave-uniform
    const bool live = w.element < p.width;
    float x[R][8];
    // rows and columns past the end read the last ones again: the requests go out before the places are known
    const int64_t stride = w.which ? p.v_rs : p.k_rs;
    const T *from = static_cast<const T *>(w.which ? p.v_in : p.k_in) + min(w.element, p.width - 8);
#pragma unroll
    for (int r = 0; r < R; ++r) load_floats<T, 8>(from + min(w.row + r, p.rows - 1) * stride, x[r]);
    w.find(p);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (__builtin_amdgcn_readlane(w.page, r) < 0) continue;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(unsigned, x[r][i]) & 0x7fffffffu);
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
        top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
        const unsigned byte = kv4_scale_byte(top);
        const float s = kv4_scale(byte);
        unsigned c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[r][0], x[r][1], s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[r][2], x[r][3], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[r][4], x[r][5], s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[r][6], x[r][7], s, 3);
        if (live) {
            uint8_t *codes, *scale;
            w.template addresses<D>(p, r, codes, scale);
            *reinterpret_cast<unsigned *>(codes) = byte == 255 ? 0u : c;
            if ((threadIdx.x & 3) == 0) *scale = (uint8_t)byte;
        }
    }
}

template <typename T, int D, int R>
__global__ __launch_bounds__(256) void gather_kernel(RowsParams p) {
    Places<R> w(p);
    if (w.row >= p.rows) return;                                 // wave-uniform
    w.find(p);
    if (w.element >= p.width) return;
    unsigned code[R], byte[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        code[r] = byte[r] = 0;
        if (__builtin_amdgcn_readlane(w.page, r) >= 0) {
            uint8_t *codes, *scale;
            w.template addresses<D>(p, r, codes, scale);
            code[r] = *reinterpret_cast<const unsigned *>(codes);
            byte[r] = *scale;
        }
    }
    const int64_t stride = w.which ? p.v_rs : p.k_rs;
    T *to = static_cast<T *>(w.which ? p.v_out : p.k_out) + w.element;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (w.row + r >= p.rows || (!(w.owned >> r & 1) && !p.zero_rest)) continue;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (__builtin_amdgcn_readlane(w.page, r) >= 0) kv4_values(code[r], byte[r], x);
        store_floats<T, 8>(to + (w.row + r) * stride, x);
    }
}

// Rows a wave takes: one where the call is short of waves, four (four requests under way, one search) from two waves for each
// of the 8192 that the card holds at once.  One / four: 4000 rows of 8 heads of 128, bf16 (16000 waves) 8.0 / 6.8 us append, 7.6 / 6.9
// gather; 64 rows of 25 heads of 64, fp32 (512) 3.0 / 3.9, 3.0 / 3.9; 8000 rows of 8 of 128 (32000) 13.4 / 11.3, 12.3 / 9.9; 60000
// rows of 2 of 64, fp16 (120000) 31.8 / 20.7, 29.6 / 18.7.  Eight rows were slower than four at 32000 waves (12.0, 10.3).
constexpr int kWaveRows = 4, kManyWaves = 16384;
template <typename T, int D> struct Kernels {
    static const void *append(bool many) { return many ? reinterpret_cast<const void *>(append_kernel<T, D, kWaveRows>) : reinterpret_cast<const void *>(append_kernel<T, D, 1>); }
    static const void *gather(bool many) { return many ? reinterpret_cast<const void *>(gather_kernel<T, D, kWaveRows>) : reinterpret_cast<const void *>(gather_kernel<T, D, 1>); }
};
template <int D>
const void *kernel_of(bool append, int dtype, bool many) {
    if (dtype == CMHSA_F32) return append ? Kernels<float, D>::append(many) : Kernels<float, D>::gather(many);
    if (dtype == CMHSA_BF16) return append ? Kernels<bf16_t, D>::append(many) : Kernels<bf16_t, D>::gather(many);
    return append ? Kernels<f16_t, D>::append(many) : Kernels<f16_t, D>::gather(many);
}

// the checks that append and gather share, and the launch
int rows_call(RowsParams p, bool append, int dtype, int64_t k_rs, int64_t v_rs, const void *k, const void *v, const int *cu, int num_seqs, int rows,
              int num_kv_heads, int head_dim, hipStream_t stream) {
    if (!k || !v || (!cu && num_seqs)) return CMHSA_ERR_NULL_POINTER;
    const int64_t size = dtype == CMHSA_F32 ? 4 : 2, width = (int64_t)num_kv_heads * head_dim;
    if (k_rs < 0 || v_rs < 0 || (rows > 1 && (k_rs < width || v_rs < width))) return CMHSA_ERR_BAD_SHAPE;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || (((k_rs | v_rs) * size) & 15) || ((uintptr_t)cu & 3) || ((uintptr_t)p.starts & 3)) return CMHSA_ERR_ALIGNMENT;
    if (width > (1 << 24) || num_seqs > 0x7fffffff - 1024) return CMHSA_ERR_TOO_LARGE;
    p.k_rs = k_rs; p.v_rs = v_rs;
    p.cu = cu; p.num_seqs = num_seqs; p.rows = rows;
    p.width = (int)width;
    p.chunks = (int)((width + 511) / 512);
    const bool many = (int64_t)rows * 2 * p.chunks >= kManyWaves;
    const int each = many ? kWaveRows : 1;
    const int64_t waves = ((int64_t)rows + each - 1) / each * 2 * p.chunks;
    if (!fits_a_launch((waves + 3) / 4, 256)) return CMHSA_ERR_TOO_LARGE;
    const void *fn = head_dim == 64 ? kernel_of<64>(append, dtype, many) : kernel_of<128>(append, dtype, many);
    void *args[] = {&p};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)((waves + 3) / 4)), dim3(256), args, 0, stream);
    return e == hipSuccess ? CMHSA_OK : (int)e;
}

bool known_type(int dtype) { return dtype == CMHSA_F32 || dtype == CMHSA_BF16 || dtype == CMHSA_F16; }

constexpr int kPairs = 440;                    // src / dst pairs a launch carries in its arguments (3520 of 4096 bytes)
constexpr int kPieceBytes = 16384;             // a workgroup's share of a page: four 16-byte pieces a thread
struct CopyParams {
    uint8_t *pages;
    int64_t layer_stride, page_stride;
    int64_t page_bytes;
    int src[kPairs], dst[kPairs];
};

__global__ __launch_bounds__(256) void copy_kernel(CopyParams p) {
    uint8_t *layer = p.pages + blockIdx.z * p.layer_stride;
    const uint8_t *from = layer + p.src[blockIdx.y] * p.page_stride;
    uint8_t *to = layer + p.dst[blockIdx.y] * p.page_stride;
    const int64_t at = (int64_t)blockIdx.x * kPieceBytes + threadIdx.x * 16;
    u32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * 4096 < p.page_bytes) x[i] = *reinterpret_cast<const u32x4 *>(from + at + i * 4096);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * 4096 < p.page_bytes) *reinterpret_cast<u32x4 *>(to + at + i * 4096) = x[i];
}

}  // namespace

extern "C" {

int cmhsa_kv4_append(const void *k, const void *v, int64_t k_row_stride, int64_t v_row_stride, int dtype,
                     uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *cu_seqlens, const int *starts, int num_seqs, int rows, int num_kv_heads, int head_dim, void *stream) {
    if (num_seqs < 0 || rows < 0 || !known_type(dtype)) return CMHSA_ERR_BAD_SHAPE;
    const int bad = kv4_check_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width, num_kv_heads, head_dim);
    if (bad) return bad;
    if (rows == 0 || num_seqs == 0) return CMHSA_OK;
    RowsParams p = {};
    p.k_in = k; p.v_in = v;
    p.pool = kv4_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width);
    p.starts = starts;
    return rows_call(p, true, dtype, k_row_stride, v_row_stride, k, v, cu_seqlens, num_seqs, rows, num_kv_heads, head_dim,
                     static_cast<hipStream_t>(stream));
}

int cmhsa_kv4_gather(void *k, void *v, int64_t k_row_stride, int64_t v_row_stride, int dtype,
                     const uint8_t *pages, int64_t page_stride, int num_pages, int page_size,
                     const int *page_table, int64_t table_stride, int table_width,
                     const int *cu_seqlens, const int *starts, int num_seqs, int rows, int num_kv_heads, int head_dim, int zero_rest, void *stream) {
    if (num_seqs < 0 || rows < 0 || !known_type(dtype)) return CMHSA_ERR_BAD_SHAPE;
    const int bad = kv4_check_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width, num_kv_heads, head_dim);
    if (bad) return bad;
    if (rows == 0 || (num_seqs == 0 && !zero_rest)) return CMHSA_OK;
    RowsParams p = {};
    p.k_out = k; p.v_out = v;
    p.pool = kv4_pool(pages, page_stride, num_pages, page_size, page_table, table_stride, table_width);
    p.starts = starts;
    p.zero_rest = zero_rest;
    return rows_call(p, false, dtype, k_row_stride, v_row_stride, k, v, cu_seqlens, num_seqs, rows, num_kv_heads, head_dim,
                     static_cast<hipStream_t>(stream));
}

int cmhsa_kv4_copy_pages(uint8_t *pages, int64_t layer_stride, int layers, int64_t page_stride, int num_pages, int64_t page_bytes,
                         const int *src, const int *dst, int count, void *stream) {
    if (layers < 0 || num_pages < 0 || count < 0 || page_bytes < 0 || page_stride < page_bytes || layer_stride < 0) return CMHSA_ERR_BAD_SHAPE;
    if (layers == 0 || count == 0 || page_bytes == 0) return CMHSA_OK;
    if (!pages || !src || !dst) return CMHSA_ERR_NULL_POINTER;
    if (((uintptr_t)pages | (uintptr_t)layer_stride | (uintptr_t)page_stride | (uintptr_t)page_bytes) & 15) return CMHSA_ERR_ALIGNMENT;
    // pages that share bytes (an overlapping view) would be copied in no order
    if (layers > 1 && num_pages > 1 && layer_stride < (num_pages - 1) * page_stride + page_bytes && page_stride < (layers - 1) * layer_stride + page_bytes) return CMHSA_ERR_BAD_SHAPE;
    if (layers > 1 && layer_stride < page_bytes) return CMHSA_ERR_BAD_SHAPE;
    if (layers > 65535 || !fits_a_launch((page_bytes + kPieceBytes - 1) / kPieceBytes, 256)) return CMHSA_ERR_TOO_LARGE;
    // a page may be read often but written once, and never both: the pairs of a call have no order
    for (int i = 0; i < count; ++i)
        if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) return CMHSA_ERR_BAD_SHAPE;
    unsigned char *mark = static_cast<unsigned char *>(calloc((size_t)num_pages, 1));
    if (!mark) return CMHSA_ERR_TOO_LARGE;
    bool clash = false;
    for (int i = 0; i < count; ++i) { clash |= mark[dst[i]] != 0; mark[dst[i]] = 1; }
    for (int i = 0; i < count; ++i) clash |= mark[src[i]] != 0;
    free(mark);
    if (clash) return CMHSA_ERR_BAD_SHAPE;
    for (int at = 0; at < count; at += kPairs) {
        CopyParams p;
        p.pages = pages; p.layer_stride = layer_stride; p.page_stride = page_stride; p.page_bytes = page_bytes;
        const int n = count - at < kPairs ? count - at : kPairs;
        for (int i = 0; i < kPairs; ++i) { p.src[i] = src[at + (i < n ? i : 0)]; p.dst[i] = dst[at + (i < n ? i : 0)]; }
        void *args[] = {&p};
        const dim3 grid((unsigned)((page_bytes + kPieceBytes - 1) / kPieceBytes), (unsigned)n, (unsigned)layers);
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(copy_kernel), grid, dim3(256), args, 0, static_cast<hipStream_t>(stream));
        if (e != hipSuccess) return (int)e;
    }
    return CMHSA_OK;
}

}  // extern "C"
