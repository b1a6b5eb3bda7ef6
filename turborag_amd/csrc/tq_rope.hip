// tq_rope.hip — per-head RMS norm and position rotation of queries and keys,
// and the same with the append of keys and values to dense pages.
//
// Mathematics, per (token, head) row x of D values, in fp32 with one rounding
// at the end:
//   y = x * w / sqrt(mean(x^2) + eps)            (a weight given; else y = x)
//   (a, b) -> (a cos - b sin, a sin + b cos)      for every pair of y
// with cos and sin of the token's position from a table.  ~7 flops a value
// against 4 bytes moved: bound by HBM, or for a decode step's few rows by the
// latency of the chain position -> table row -> result.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tq_device.h"

namespace tq {
namespace {

using namespace dev;

constexpr int kBlock = 256;

// Workgroups lie in lines of at most kLine along y: a grid has less than 2^32
// threads in x, and rows of eight million workgroups or more are 17 GB of heads.
constexpr unsigned kLine = 1u << 23;
__device__ __forceinline__ unsigned block_of() { return blockIdx.y * gridDim.x + blockIdx.x; }
dim3 grid_of(long long blocks) {
    const unsigned x = (unsigned)std::min<long long>(blocks, kLine);
    return dim3(x, (unsigned)((blocks + x - 1) / x));
}

struct RopeArgs {
    const uint16_t *q, *k, *v;   // q null: keys and values only; v null: no append
    const uint16_t *qw, *kw;     // norm weights or null
    const float* table;          // [max_position, rot]
    const int32_t *pos, *slots;
    uint16_t *oq, *ok;           // ok unused by the append
    uint8_t* pool;
    int64_t qs, ks, vs, oqs, oks;  // token strides in elements
    DenseGeom g;
    int n, hq, rows;             // tokens, query heads worked on, rows per token
    int rot, max_position;
    float eps;
};

template <bool BF>
__device__ __forceinline__ float to_float(uint16_t x) {
    return BF ? __uint_as_float((uint32_t)x << 16) : h2f(x);
}
// fp32 -> bf16 or fp16, to nearest even.
template <bool BF>
__device__ __forceinline__ uint16_t from_float(float f) {
    if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return f2h(f);
}

// Row r of a token: query head r, then key head r - hq, then value head.
// (what: 0 query, 1 key, 2 value)
struct Row {
    const uint16_t* src;
    uint16_t* dst;  // null: not stored
    const uint16_t* w;
    int what;
};
__device__ __forceinline__ Row row_of(const RopeArgs& a, int t, int r, int slot) {
    const int D = a.g.D;
    if (r < a.hq) return {a.q + t * a.qs + r * D, a.oq + t * a.oqs + r * D, a.qw, 0};
    r -= a.hq;
    const bool val = r >= a.g.H;
    if (val) r -= a.g.H;
    Row o;
    o.what = val ? 2 : 1;
    o.src = val ? a.v + t * a.vs + r * D : a.k + t * a.ks + r * D;
    o.w = val ? nullptr : a.kw;
    if (!a.v) {
        o.dst = a.ok + t * a.oks + r * D;
    } else if (slot < 0) {
        o.dst = nullptr;
    } else {
        const int page = slot / a.g.block_size, tib = slot - page * a.g.block_size;
        o.dst = reinterpret_cast<uint16_t*>(a.pool + (size_t)page * a.g.page_size +
                                            (val ? a.g.v_off : a.g.k_off)) +
                (size_t)(tib * a.g.H + r) * D;
    }
    return o;
}

// ---------------------------------------------------------------------------
// Any head_dim, rotated part and alignment: D/2 lanes per row, two values per
// lane.  Lane i < rot/2 holds pair i, the others two values that pass.
// ---------------------------------------------------------------------------
template <bool BF>
__global__ __launch_bounds__(kBlock) void rope_pairs_kernel(const RopeArgs a, int interleaved) {
    const int D = a.g.D, L = D / 2, half = a.rot / 2;
    const int i = threadIdx.x & (L - 1);
    const long long row = (long long)block_of() * (kBlock / L) + threadIdx.x / L;
    const long long all = (long long)a.n * a.rows;
    const bool valid = row < all;
    const long long rr = valid ? row : all - 1;
    const int t = (int)(rr / a.rows), r = (int)(rr - (long long)t * a.rows);
    const int pos = a.pos[t];
    const bool inside = pos >= 0 && pos < a.max_position;
    const Row o = row_of(a, t, r, a.v ? a.slots[t] : 0);
    const bool turned = i < half;
    const int e0 = !turned || interleaved ? 2 * i : i;
    const int e1 = !turned || interleaved ? 2 * i + 1 : i + half;
    const uint16_t x0 = o.src[e0], x1 = o.src[e1];
    float y0 = to_float<BF>(x0), y1 = to_float<BF>(x1);
    float ss = fmaf(y0, y0, y1 * y1);
    for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m, 64);
    if (!valid || !inside || !o.dst) return;
    if (o.what == 2) {
        o.dst[e0] = x0;
        o.dst[e1] = x1;
        return;
    }
    if (o.w) {
        const float s = 1.0f / sqrtf(ss / (float)D + a.eps);
        y0 = y0 * s * to_float<BF>(o.w[e0]);
        y1 = y1 * s * to_float<BF>(o.w[e1]);
    }
    if (turned) {
        const float* tr = a.table + (size_t)pos * a.rot + i;
        const float c = tr[0], s = tr[half];
        const float u = fmaf(y0, c, -(y1 * s));
        y1 = fmaf(y0, s, y1 * c);
        y0 = u;
    }
    o.dst[e0] = from_float<BF>(y0);
    o.dst[e1] = from_float<BF>(y1);
}

// ---------------------------------------------------------------------------
// head_dim 64 and 128, all of it rotated, 16-byte aligned rows: D / 16 lanes
// per row, each with eight pairs, so that the rotation needs no exchange: the
// two 16-byte pieces 8j .. 8j + 7 and D/2 + 8j .. of its row, or (interleaved)
// 16j .. 16j + 15; cos and sin are 8j .. 8j + 7 of the table's row either way.
// One row per lane group: a table row is as many bytes as two rows of heads,
// but a token's rows find it in the caches; two, four and five rows per group
// with the table row in registers took 66 to 69 us against 66 for the append
// of 32,768 tokens of 16/2 heads (352 MB: 5.3 TB/s; a copy of 1 GiB runs at 5.2),
// and 3.7 to 4.7 against 3.4 for 1,143 tokens of 14/2 heads at head_dim 64.
// ---------------------------------------------------------------------------
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <bool BF>
__device__ __forceinline__ void unpack8(u4 w, float* y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[2 * e] = to_float<BF>(w[e] & 0xffff);
        y[2 * e + 1] = to_float<BF>(w[e] >> 16);
    }
}
template <bool BF>
__device__ __forceinline__ u4 pack8(const float* y) {
    u4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (BF) {
            typedef float f2v __attribute__((ext_vector_type(2)));
            typedef __bf16 b2v __attribute__((ext_vector_type(2)));
            w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){y[2 * e], y[2 * e + 1]}, b2v));
        } else {
            w[e] = f2h2(y[2 * e], y[2 * e + 1]);
        }
    }
    return w;
}

template <bool BF, int D, bool INTER>
__global__ __launch_bounds__(kBlock) void rope_rows_kernel(const RopeArgs a) {
    constexpr int L = D / 16;
    const int j = threadIdx.x & (L - 1);
    const int job = block_of() * (kBlock / L) + threadIdx.x / L;
    const int row = min(job, a.n * a.rows - 1);
    const int t = row / a.rows;
    const int pos = a.pos[t], slot = a.v ? a.slots[t] : 0;
    const Row o = row_of(a, t, row - t * a.rows, slot);
    const int at0 = INTER ? 16 * j : 8 * j, at1 = INTER ? 16 * j + 8 : D / 2 + 8 * j;
    u4 w0 = *reinterpret_cast<const u4*>(o.src + at0), w1 = *reinterpret_cast<const u4*>(o.src + at1);
    const bool live = job == row && pos >= 0 && pos < a.max_position && o.dst;
    if (o.what != 2) {  // (the same for a row's lanes)
        const float* tr = a.table + (size_t)(live ? pos : 0) * D + 8 * j;
        float c[8], s[8], y[16];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<f4*>(c + e) = *reinterpret_cast<const f4*>(tr + e);
            *reinterpret_cast<f4*>(s + e) = *reinterpret_cast<const f4*>(tr + D / 2 + e);
        }
        unpack8<BF>(w0, y);
        unpack8<BF>(w1, y + 8);
        if (o.w) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) ss = fmaf(y[e], y[e], ss);
            ss += quad_xor<1>(ss);
            ss += quad_xor<2>(ss);
            if (L == 8)  // every lane of a quad holds its sum: the row's other quad by mirror
                ss += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(ss), 0x141, 0xF, 0xF, true));
            const float n = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
            float w[16];
            unpack8<BF>(*reinterpret_cast<const u4*>(o.w + at0), w);
            unpack8<BF>(*reinterpret_cast<const u4*>(o.w + at1), w + 8);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = y[e] * n * w[e];
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int i0 = INTER ? 2 * p : p, i1 = INTER ? 2 * p + 1 : p + 8;
            const float u = y[i0], v = y[i1];
            y[i0] = fmaf(u, c[p], -(v * s[p]));
            y[i1] = fmaf(u, s[p], v * c[p]);
        }
        w0 = pack8<BF>(y);
        w1 = pack8<BF>(y + 8);
    }
    if (live) {
        *reinterpret_cast<u4*>(o.dst + at0) = w0;
        *reinterpret_cast<u4*>(o.dst + at1) = w1;
    }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows, weights and cells of whole 16-byte pieces.
bool rows_ok(const RopeArgs& a) {
    if ((a.g.D != 64 && a.g.D != 128) || a.rot != a.g.D) return false;
    const auto stride_ok = [&](int64_t st) { return a.n == 1 || (st & 7) == 0; };
    if (!al16(a.q) || !al16(a.k) || !al16(a.v) || !al16(a.oq) || !al16(a.ok) || !al16(a.qw) ||
        !al16(a.kw) || !al16(a.table) || !al16(a.pool))
        return false;
    if (!stride_ok(a.qs) || !stride_ok(a.ks) || !stride_ok(a.vs) || !stride_ok(a.oqs) || !stride_ok(a.oks))
        return false;
    return !a.v || ((a.g.page_size | a.g.k_off | a.g.v_off) & 15) == 0;
}

template <bool BF, int D, bool INTER>
void launch_rows(const RopeArgs& a, hipStream_t stream) {
    constexpr int per = kBlock / (D / 16);
    const dim3 grid = grid_of(((long long)a.n * a.rows + per - 1) / per);
    hipLaunchKernelGGL((rope_rows_kernel<BF, D, INTER>), grid, dim3(kBlock), 0, stream, a);
}

void launch_rope(const RopeArgs& a, bool bf16, bool interleaved, hipStream_t stream) {
    if (a.n == 0 || a.rows == 0) return;
    const char* what = a.v ? "dense_rope_append_kv_kernel" : "qk_norm_rope_kernel";
    if (rows_ok(a)) {
        const auto go = [&](auto bf, auto inter) {
            constexpr bool BF = decltype(bf)::value, IN = decltype(inter)::value;
            a.g.D == 128 ? launch_rows<BF, 128, IN>(a, stream) : launch_rows<BF, 64, IN>(a, stream);
        };
        if (bf16)
            interleaved ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
        else
            interleaved ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
        check_launch(what);
        return;
    }
    const int per = kBlock / (a.g.D / 2);
    const long long rows = (long long)a.n * a.rows;
    const dim3 grid = grid_of((rows + per - 1) / per);
    if (bf16)
        hipLaunchKernelGGL(rope_pairs_kernel<true>, grid, dim3(kBlock), 0, stream, a, (int)interleaved);
    else
        hipLaunchKernelGGL(rope_pairs_kernel<false>, grid, dim3(kBlock), 0, stream, a, (int)interleaved);
    check_launch(what);
}

// Checks shared by both entries; fills what does not depend on the pages.
void check_rope(const char* what, const TQRopeConfig& r, const TQConfig& cfg, int num_tokens) {
    const std::string w = std::string(what) + ": ";
    const int D = cfg.head_dim;
    if (D < 2 || D > 128 || (D & (D - 1)))
        throw Error(w + "head_dim must be a power of two in [2, 128]");
    if (cfg.num_kv_heads <= 0) throw Error(w + "num_kv_heads must be > 0");
    if (r.num_q_heads <= 0) throw Error(w + "num_q_heads must be > 0");
    if (r.dtype != TQ_DTYPE_FP16 && r.dtype != TQ_DTYPE_BF16)
        throw Error(w + "dtype must be TQ_DTYPE_FP16 or TQ_DTYPE_BF16");
    if (r.rot_dim < 2 || r.rot_dim > D || (r.rot_dim & 1))
        throw Error(w + "rot_dim must be even in [2, head_dim]");
    if (r.max_position <= 0) throw Error(w + "max_position must be > 0");
    if (!(r.eps >= 0.0f)) throw Error(w + "eps must be >= 0");
    if (num_tokens < 0) throw Error(w + "num_tokens must be >= 0");
    if ((long long)num_tokens * ((long long)r.num_q_heads + 2LL * cfg.num_kv_heads) >= (1LL << 30))
        throw Error(w + "num_tokens * heads must be < 2^30");
}

void check_rows(const char* what, const char* name, const void* p, int64_t stride, int heads, int D,
                int num_tokens) {
    if (reinterpret_cast<uintptr_t>(p) & 1)
        throw Error(std::string(what) + ": " + name + " must be 2-byte aligned");
    if (num_tokens > 1 && (stride < (int64_t)heads * D || stride >= (int64_t(1) << 40)))
        throw Error(std::string(what) + ": " + name + " token stride must be at least heads * head_dim");
}

template <class F>
int rope_entry(void* stream, F&& f) {
    try {
        f();
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

extern "C" int tq_launch_qk_norm_rope(const void* query, int64_t query_stride, const void* key,
                                      int64_t key_stride, const void* q_weight,
                                      const void* k_weight, const float* cos_sin,
                                      const int32_t* positions, void* out_query,
                                      int64_t out_query_stride, void* out_key,
                                      int64_t out_key_stride, const TQRopeConfig* rope,
                                      const TQConfig* cfg, int num_tokens, void* stream) {
    if (!query || !key || !cos_sin || !positions || !out_query || !out_key || !rope || !cfg) return -1;
    return tq::rope_entry(stream, [&] {
        const char* what = "qk_norm_rope";
        tq::check_rope(what, *rope, *cfg, num_tokens);
        const int H = cfg->num_kv_heads, D = cfg->head_dim, Hq = rope->num_q_heads;
        tq::check_rows(what, "query", query, query_stride, Hq, D, num_tokens);
        tq::check_rows(what, "key", key, key_stride, H, D, num_tokens);
        tq::check_rows(what, "out_query", out_query, out_query_stride, Hq, D, num_tokens);
        tq::check_rows(what, "out_key", out_key, out_key_stride, H, D, num_tokens);
        tq::RopeArgs a{};
        a.q = static_cast<const uint16_t*>(query);
        a.k = static_cast<const uint16_t*>(key);
        a.qw = static_cast<const uint16_t*>(q_weight);
        a.kw = static_cast<const uint16_t*>(k_weight);
        a.table = cos_sin;
        a.pos = positions;
        a.oq = static_cast<uint16_t*>(out_query);
        a.ok = static_cast<uint16_t*>(out_key);
        a.qs = query_stride;
        a.ks = key_stride;
        a.oqs = out_query_stride;
        a.oks = out_key_stride;
        a.g.H = H;
        a.g.D = D;
        a.g.block_size = 1;
        a.n = num_tokens;
        a.hq = Hq;
        a.rows = Hq + H;
        a.rot = rope->rot_dim;
        a.max_position = rope->max_position;
        a.eps = rope->eps;
        tq::launch_rope(a, rope->dtype == TQ_DTYPE_BF16, rope->interleaved != 0,
                        static_cast<hipStream_t>(stream));
    });
}

extern "C" int tq_launch_dense_rope_append_kv(
    const void* query, int64_t query_stride, const void* key, int64_t key_stride, const void* value,
    int64_t value_stride, const void* q_weight, const void* k_weight, const float* cos_sin,
    const int32_t* positions, const int32_t* slot_mapping, uint8_t* page_pool, void* out_query,
    int64_t out_query_stride, const TQDensePageLayout* layout, const TQRopeConfig* rope,
    const TQConfig* cfg, int num_tokens, void* stream) {
    if (!key || !value || !cos_sin || !positions || !slot_mapping || !page_pool || !layout || !rope ||
        !cfg || !query != !out_query)
        return -1;
    return tq::rope_entry(stream, [&] {
        const char* what = "dense_rope_append_kv";
        tq::check_rope(what, *rope, *cfg, num_tokens);
        const int H = cfg->num_kv_heads, D = cfg->head_dim, Hq = query ? rope->num_q_heads : 0;
        tq::RopeArgs a{};
        a.g = tq::dense_geom(*cfg, *layout);
        for (const uint64_t off : {a.g.k_off, a.g.v_off})
            if (off > a.g.page_size || layout->k_bytes > a.g.page_size - off)
                throw tq::Error("dense_rope_append_kv: layout does not match cfg (a region ends past the page)");
        if (reinterpret_cast<uintptr_t>(page_pool) & 3)
            throw tq::Error("dense_rope_append_kv: page_pool must be 4-byte aligned");
        if (query) {
            tq::check_rows(what, "query", query, query_stride, Hq, D, num_tokens);
            tq::check_rows(what, "out_query", out_query, out_query_stride, Hq, D, num_tokens);
        }
        tq::check_rows(what, "key", key, key_stride, H, D, num_tokens);
        tq::check_rows(what, "value", value, value_stride, H, D, num_tokens);
        a.q = static_cast<const uint16_t*>(query);
        a.k = static_cast<const uint16_t*>(key);
        a.v = static_cast<const uint16_t*>(value);
        a.qw = static_cast<const uint16_t*>(q_weight);
        a.kw = static_cast<const uint16_t*>(k_weight);
        a.table = cos_sin;
        a.pos = positions;
        a.slots = slot_mapping;
        a.pool = page_pool;
        a.oq = static_cast<uint16_t*>(out_query);
        a.qs = query_stride;
        a.ks = key_stride;
        a.vs = value_stride;
        a.oqs = out_query_stride;
        a.n = num_tokens;
        a.hq = Hq;
        a.rows = Hq + 2 * H;
        a.rot = rope->rot_dim;
        a.max_position = rope->max_position;
        a.eps = rope->eps;
        tq::launch_rope(a, rope->dtype == TQ_DTYPE_BF16, rope->interleaved != 0,
                        static_cast<hipStream_t>(stream));
    });
}
