// tq_tree.hip — attention of drafted token trees over paged caches: dense
// pages (fp16, bf16), turbo_prod and turbo_mse pages.
//
// Row (token r of sequence s, query head) attends the tokens t of s with
// t < prefix_len[s], or t = prefix_len[s] + j with bit j of the row's mask:
//   out = sum_t softmax_t(<q, k_t> / sqrt(D)) v_t.
// Compressed pages hold k and v rotated (an orthogonal transform), so q is
// rotated the same way, and the output rotated back.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tq_device.h"

namespace tq {
namespace {

using namespace dev;

// What the pages hold.
constexpr int kFp16 = 0, kBf16 = 1, kProd = 2, kMse = 3;

struct TreeArgs {
    const uint16_t* query;
    const uint8_t* pool;
    const int32_t *tables, *row_start, *prefix, *mask;
    uint16_t* out;
    PageGeom g;  // dense pages: kc_off, vc_off and code_stride of fp16/bf16 rows
    int max_blocks, mask_words, hq, seqs, tokens, max_kv;
};

template <bool BF>
__device__ __forceinline__ float to_float(uint16_t x) {
    return BF ? __uint_as_float((uint32_t)x << 16) : h2f(x);
}
template <bool BF>
__device__ __forceinline__ uint16_t from_float(float f) {
    if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return f2h(f);
}

// Element d of a cell's K or V row.
template <int FMT>
__device__ float cell_value(const TreeArgs& a, const uint8_t* page, int cell, int d, bool key) {
    const PageGeom& g = a.g;
    const uint8_t* row = page + (key ? g.kc_off : g.vc_off) + (size_t)cell * g.code_stride;
    if constexpr (FMT == kFp16 || FMT == kBf16) return to_float<FMT == kBf16>(ld_u16(row + 2 * d));
    const int n = (row[d >> 1] >> (4 * (d & 1))) & 15;
    const float s = h2f(ld_u16(page + (key ? g.ks_off : g.vs_off) + (size_t)cell * 2));
    if (FMT == kProd && key) {
        const float e = h2f(ld_u16(page + g.kres_off + (size_t)cell * 2));
        return (pick(kK3, n & 7) + (n & 8 ? e : -e)) * s;
    }
    return pick(kV4, n) * s;
}

// One wave per (row, query head).
template <int FMT, int D>
__global__ __launch_bounds__(64) void tree_rows_kernel(const TreeArgs a, float inv) {
    __shared__ float q[D];
    const int r = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x;
    const int h = hq / (a.hq / a.g.H);
    // The row's sequence: the starts are non-decreasing.
    int s = 0;
    for (int b = 0; b < a.seqs; b += 64)
        s += __popcll(__ballot(b + lane < a.seqs && a.row_start[1 + b + lane] <= r));
    if (s >= a.seqs || r < a.row_start[s]) return;
    const int n = min(a.row_start[s + 1], a.tokens) - a.row_start[s];
    const int L = max(a.prefix[s], 0);
    const int end = (int)min((long long)L + n, (long long)a.max_kv);
    constexpr bool turned = FMT == kProd || FMT == kMse, BF = FMT == kBf16;
    auto rotate = [&] {  // q = WHT(q) / sqrt(D), lane pairs through LDS
        for (int m = 1; m < D; m <<= 1) {
            __syncthreads();
            for (int i = lane; i < D / 2; i += 64) {
                const int lo = (i / m) * 2 * m + i % m;
                const float u = q[lo], w = q[lo + m];
                q[lo] = u + w;
                q[lo + m] = u - w;
            }
        }
        __syncthreads();
        for (int d = lane; d < D; d += 64) q[d] *= inv;
    };
    const size_t ro = ((size_t)r * a.hq + hq) * D;
    for (int d = lane; d < D; d += 64)
        q[d] = to_float<BF>(a.query[ro + d]) * (turned ? sign_of(d, h) : 1.0f);
    if (turned) rotate();
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[D / 64] = {};
    for (int t0 = 0; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        bool seen = t < end;
        if (seen && t >= L) {
            const int j = t - L;
            seen = j < 32 * a.mask_words && (a.mask[(size_t)r * a.mask_words + (j >> 5)] >> (j & 31) & 1);
        }
        int id = -1;
        if (seen) id = a.tables[(size_t)s * a.max_blocks + t / a.g.block_size];
        seen = seen && id >= 0;
        const uint8_t* page = a.pool + (size_t)max(id, 0) * a.g.page_size;
        const int cell = (t % a.g.block_size) * a.g.H + h;
        float x = -INFINITY;
        if (seen) {
            x = 0.0f;
            for (int d = 0; d < D; ++d) x = fmaf(q[d], cell_value<FMT>(a, page, cell, d, true), x);
            x *= inv;
        }
        const float mn = fmaxf(m, max_lanes<64>(x));
        const float p = seen ? expf(x - mn) : 0.0f, f = mn == -INFINITY ? 1.0f : expf(m - mn);
        l = l * f + sum_lanes<64>(p);
        m = mn;
        for (int i = 0; i < D / 64; ++i) o[i] *= f;
        const unsigned long long all = __ballot(seen);
        for (int k = 0; k < 64; ++k) {
            if (!(all >> k & 1)) continue;
            const float pk = __shfl(p, k);
            const uint8_t* pg = a.pool + (size_t)__shfl(id, k) * a.g.page_size;
            const int c = __shfl(cell, k);
            for (int i = 0; i < D / 64; ++i)
                o[i] = fmaf(pk, cell_value<FMT>(a, pg, c, lane + 64 * i, false), o[i]);
        }
    }
    __syncthreads();
    for (int i = 0; i < D / 64; ++i) q[lane + 64 * i] = l == 0.0f ? 0.0f : o[i] / l;
    if (turned) rotate();
    __syncthreads();
    for (int d = lane; d < D; d += 64)
        a.out[ro + d] = from_float<BF>(q[d] * (turned ? sign_of(d, h) : 1.0f));
}

void launch_tree(int fmt, const TreeArgs& a, hipStream_t stream) {
    const dim3 grid(a.tokens, a.hq);
    const float inv = inv_sqrt_d(a.g.D);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(64), 0, stream, a, inv);
        check_launch("tree_attention_kernel");
    };
    if (a.g.D == 128) {
        switch (fmt) {
            case kFp16: return go(tree_rows_kernel<kFp16, 128>);
            case kBf16: return go(tree_rows_kernel<kBf16, 128>);
            case kProd: return go(tree_rows_kernel<kProd, 128>);
            default: return go(tree_rows_kernel<kMse, 128>);
        }
    }
    switch (fmt) {
        case kFp16: return go(tree_rows_kernel<kFp16, 64>);
        case kBf16: return go(tree_rows_kernel<kBf16, 64>);
        case kProd: return go(tree_rows_kernel<kProd, 64>);
        default: return go(tree_rows_kernel<kMse, 64>);
    }
}

bool aligned(uint64_t v, uint64_t a) { return (v & (a - 1)) == 0; }
bool aligned(const void* p, uint64_t a) { return aligned(reinterpret_cast<uintptr_t>(p), a); }

PageGeom dense_rows(const TQConfig& cfg, const TQDensePageLayout& l) {
    const DenseGeom d = dense_geom(cfg, l);
    PageGeom g{};
    g.page_size = d.page_size;
    g.kc_off = d.k_off;
    g.vc_off = d.v_off;
    g.code_stride = 2 * d.D;
    g.H = d.H;
    g.D = d.D;
    g.block_size = d.block_size;
    g.bs_shift = (d.block_size & (d.block_size - 1)) == 0 ? __builtin_ctz(d.block_size) : -1;
    return g;
}

template <class Geom>
int tree_entry(const char* name, int fmt, Geom&& geom, const void* query, const uint8_t* pool,
               const int32_t* tables, int max_blocks, const int32_t* row_start,
               const int32_t* prefix, const int32_t* mask, int mask_words, void* output, int hq,
               int seqs, int tokens, int max_kv, void* stream) {
    try {
        const std::string w = std::string(name) + ": ";
        TreeArgs a{};
        a.g = geom();
        const PageGeom& g = a.g;
        if (g.D != 64 && g.D != 128) throw Error(w + "head_dim must be 64 or 128");
        if (hq <= 0 || hq % g.H || hq > 65535)
            throw Error(w + "num_q_heads must be a multiple of num_kv_heads, at most 65535");
        if (seqs < 0 || tokens < 0) throw Error(w + "num_seqs and num_tokens must be >= 0");
        if (max_blocks <= 0 || mask_words <= 0)
            throw Error(w + "max_blocks_per_seq and mask_words must be > 0");
        if (max_kv < 0 || max_kv > (1 << 30) || (long long)max_blocks * g.block_size < max_kv)
            throw Error(w + "max_kv_len must be in [0, 2^30] and fit in max_blocks_per_seq pages");
        if ((long long)tokens * hq >= (1LL << 26))
            throw Error(w + "num_tokens * num_q_heads must be < 2^26");
        const uint64_t al = fmt <= kBf16 ? 16 : 2;
        if (!aligned(pool, al) || !aligned(g.page_size | g.kc_off | g.vc_off, al) ||
            !aligned(g.ks_off | g.kres_off | g.vs_off, 2))
            throw Error(w + (al == 16 ? "page_pool, page size and offsets must be 16-byte aligned"
                                      : "page_pool, page size and offsets must be 2-byte aligned"));
        if (!aligned(query, 16) || !aligned(output, 16))
            throw Error(w + "query and output must be 16-byte aligned");
        if (seqs == 0 || tokens == 0) return 0;
        a.query = static_cast<const uint16_t*>(query);
        a.pool = pool;
        a.tables = tables;
        a.row_start = row_start;
        a.prefix = prefix;
        a.mask = mask;
        a.out = static_cast<uint16_t*>(output);
        a.max_blocks = max_blocks;
        a.mask_words = mask_words;
        a.hq = hq;
        a.seqs = seqs;
        a.tokens = tokens;
        a.max_kv = max_kv;
        launch_tree(fmt, a, static_cast<hipStream_t>(stream));
        debug_sync(stream);
        return 0;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return -2;
    } catch (...) {
        set_last_error("unknown error");
        return -2;
    }
}

}  // namespace
}  // namespace tq

extern "C" int tq_launch_dense_tree_attention(
    const void* query, const uint8_t* page_pool, const int32_t* block_tables,
    int max_blocks_per_seq, const int32_t* row_start, const int32_t* prefix_len,
    const int32_t* tree_mask, int mask_words, void* output, const TQDensePageLayout* layout,
    const TQConfig* cfg, int dtype, int num_q_heads, int num_seqs, int num_tokens, int max_kv_len,
    void* stream) {
    if (!query || !page_pool || !block_tables || !row_start || !prefix_len || !tree_mask || !output ||
        !layout || !cfg)
        return -1;
    return tq::tree_entry(
        "dense_tree_attention", dtype == TQ_DTYPE_BF16 ? tq::kBf16 : tq::kFp16,
        [&] {
            if (dtype != TQ_DTYPE_FP16 && dtype != TQ_DTYPE_BF16)
                throw tq::Error("dense_tree_attention: dtype must be TQ_DTYPE_FP16 or TQ_DTYPE_BF16");
            return tq::dense_rows(*cfg, *layout);
        },
        query, page_pool, block_tables, max_blocks_per_seq, row_start, prefix_len, tree_mask,
        mask_words, output, num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}

extern "C" int tq_launch_turbo_prod_tree_attention(
    const uint16_t* query, const uint8_t* page_pool, const int32_t* block_tables,
    int max_blocks_per_seq, const int32_t* row_start, const int32_t* prefix_len,
    const int32_t* tree_mask, int mask_words, uint16_t* output,
    const TQTurboProdPageLayout* layout, const TQConfig* cfg, int num_q_heads, int num_seqs,
    int num_tokens, int max_kv_len, void* stream) {
    if (!query || !page_pool || !block_tables || !row_start || !prefix_len || !tree_mask || !output ||
        !layout || !cfg)
        return -1;
    return tq::tree_entry(
        "turbo_prod_tree_attention", tq::kProd, [&] { return tq::prod_geom(*cfg, *layout); }, query,
        page_pool, block_tables, max_blocks_per_seq, row_start, prefix_len, tree_mask, mask_words,
        output, num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}

extern "C" int tq_launch_turbo_mse_tree_attention(
    const uint16_t* query, const uint8_t* page_pool, const int32_t* block_tables,
    int max_blocks_per_seq, const int32_t* row_start, const int32_t* prefix_len,
    const int32_t* tree_mask, int mask_words, uint16_t* output, const TQTurbomsePageLayout* layout,
    const TQConfig* cfg, int num_q_heads, int num_seqs, int num_tokens, int max_kv_len,
    void* stream) {
    if (!query || !page_pool || !block_tables || !row_start || !prefix_len || !tree_mask || !output ||
        !layout || !cfg)
        return -1;
    return tq::tree_entry(
        "turbo_mse_tree_attention", tq::kMse, [&] { return tq::mse_geom(*cfg, *layout); }, query,
        page_pool, block_tables, max_blocks_per_seq, row_start, prefix_len, tree_mask, mask_words,
        output, num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}
