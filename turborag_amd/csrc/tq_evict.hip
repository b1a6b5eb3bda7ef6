// tq_evict.hip — eviction from paged caches: the tokens that a budget keeps, by their
// scores, and the move of their cells to the front.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tq_device.h"

namespace tq {
namespace {

using namespace dev;

// ---------------------------------------------------------------------------
// Selection.  One workgroup per (sequence, kv head): a radix search of the lowest kept
// score over the bits of an order-preserving key, three digits of 11, 11 and 10 bits,
// counted in LDS; then the kept tokens in order, their places from counts of each wave's
// stretch of tokens.  4 bytes a token and pass: bound by the latency of the passes.
// ---------------------------------------------------------------------------
struct SelectArgs {
    const float* scores;
    int64_t stride, out_stride;  // from one head's scores to the next
    const int32_t* kv_len;
    int32_t *kept, *new_len;  // new_len or null
    float* out;               // null, or the kept tokens' scores; may be the scores
    int heads, max_kv, budget, sink, recent;
};

// Larger scores have larger keys; -0 is 0, NaN is below everything.
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);
    return f != f ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kWaves = 16, kThreads = 64 * kWaves, kBins = 2048;

__global__ __launch_bounds__(kThreads) void select_kv_kernel(const SelectArgs a) {
    __shared__ uint32_t bins[kBins];
    __shared__ uint32_t above[kWaves], found[2];
    __shared__ int2 counts[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x;
    const int s = (int)(row / a.heads), B = a.budget;
    const int L = min(max(a.kv_len[s], 0), a.max_kv), n = min(L, B);
    const float* x = a.scores + row * a.stride;
    int32_t* kept = a.kept + row * B;
    float* out = a.out ? a.out + row * a.out_stride : nullptr;
    if (a.new_len && row == (int64_t)s * a.heads && tid == 0) a.new_len[s] = n;
    for (int j = n + tid; j < B; j += kThreads) kept[j] = -1;

    if (L <= B) {
        for (int j = tid; j < L; j += kThreads) kept[j] = j;
        if (out && out != x)
            for (int j = tid; j < L; j += kThreads) out[j] = x[j];
    } else {
        // [lo, hi): the tokens that their scores decide on.
        const int lo = a.sink, hi = L - a.recent;
        uint32_t want = (uint32_t)(B - a.sink - a.recent), prefix = 0;
        int shift = 32;
        if (want) {
            for (int pass = 0; pass < 3; ++pass) {
                const int bits = pass < 2 ? 11 : 10, from = shift;
                shift -= bits;
                const uint32_t top = (1u << bits) - 1;
                for (int k = tid; k < kBins; k += kThreads) bins[k] = 0;
                __syncthreads();
                for (int t = lo + tid; t < hi; t += kThreads) {
                    const uint32_t key = key_of(x[t]);
                    if (from == 32 || key >> from == prefix) atomicAdd(&bins[key >> shift & top], 1u);
                }
                __syncthreads();
                // The digit at which the tokens from the top reach `want`: a wave has 128
                // bins, a lane two of them (from the top).
                const int d1 = kBins - 1 - 2 * tid, d0 = d1 - 1;
                const uint32_t n1 = bins[d1], n0 = bins[d0];
                uint32_t up = n1 + n0;
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const uint32_t o = __shfl_up(up, m, 64);
                    if (lane >= m) up += o;
                }
                if (lane == 63) above[wv] = up;
                __syncthreads();
                uint32_t before = up - n1 - n0;
                for (int w = 0; w < wv; ++w) before += above[w];
                if (before < want && before + n1 >= want) {
                    found[0] = (uint32_t)d1;
                    found[1] = want - before;
                } else if (before + n1 < want && before + n1 + n0 >= want) {
                    found[0] = (uint32_t)d0;
                    found[1] = want - before - n1;
                }
                __syncthreads();
                prefix = prefix << bits | found[0];
                want = found[1];
                __syncthreads();
            }
        }
        // prefix: the lowest kept key; `want` tokens with it are kept, the first ones.
        const bool none = a.sink + a.recent == B;
        const int per = ((L + kWaves - 1) / kWaves + 63) & ~63, t0 = min(wv * per, L), t1 = min(t0 + per, L);
        const auto look = [&](int t, bool& sure, bool& tie) {
            const bool in = t < t1;
            const uint32_t key = in ? key_of(x[t]) : 0u;
            const bool mid = t >= lo && t < hi;
            sure = in && (!mid || (!none && key > prefix));
            tie = in && mid && !none && key == prefix;
        };
        int sure_n = 0, tie_n = 0;
        for (int t = t0; t < t1; t += 64) {
            bool sure, tie;
            look(t + lane, sure, tie);
            sure_n += __popcll(__ballot(sure));
            tie_n += __popcll(__ballot(tie));
        }
        if (lane == 0) counts[wv] = make_int2(sure_n, tie_n);
        __syncthreads();
        int at = 0, ties = 0;  // kept tokens and ties before the wave's
        for (int w = 0; w < wv; ++w) {
            at += counts[w].x;
            ties += counts[w].y;
        }
        at += min(ties, (int)want);
        const uint64_t below = (1ull << lane) - 1;
        for (int t = t0; t < t1; t += 64) {
            bool sure, tie;
            look(t + lane, sure, tie);
            const uint64_t tm = __ballot(tie);
            const bool keep = sure || (tie && ties + __popcll(tm & below) < (int)want);
            const uint64_t km = __ballot(keep);
            if (keep) kept[at + __popcll(km & below)] = t + lane;
            at += __popcll(km);
            ties += __popcll(tm);
        }
        if (out) {
            // In order, so that in place no score is overwritten before it is read: place j
            // takes the score of a token at j or behind it.
            __threadfence_block();
            __syncthreads();
            constexpr int kDeep = 4;
            for (int j0 = 0; j0 < n; j0 += kDeep * kThreads) {
                float v[kDeep];
#pragma unroll
                for (int k = 0; k < kDeep; ++k) {
                    const int j = j0 + k * kThreads + tid;
                    v[k] = j < n ? x[kept[j]] : 0.0f;
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < kDeep; ++k) {
                    const int j = j0 + k * kThreads + tid;
                    if (j < n) out[j] = v[k];
                }
            }
        }
    }
    if (out) {
        __syncthreads();
        for (int j = n + tid; j < a.max_kv; j += kThreads) out[j] = 0.0f;
    }
}

// ---------------------------------------------------------------------------
// Compaction.  A cell is copied in 16-byte units (its K, its V) and, for compressed
// pages, its 16-bit scales; every byte is read once and written once: bound by HBM.
// A workgroup has a chunk of kept tokens of one (sequence, kv head), whole in registers
// between its reads and its writes.
//
// In place, chunk c's places [a, b) may hold tokens that other chunks keep.  Kept token
// j comes from a place >= j, so those are chunks before c: a workgroup says when its
// reads are done, and waits with its writes for the chunks before it.  Chunks are taken
// by tickets in that order, so what a workgroup waits for has begun, and reads wait for
// nothing: every wait ends, whatever runs beside.
// ---------------------------------------------------------------------------
struct CompactArgs {
    uint8_t* pool;
    const int32_t *tables, *out_tables, *kept;
    int max_blocks, out_max_blocks, budget, chunks;
    uint64_t page_size;
    uint64_t unit_off[2], scale_off[3];  // K, V; scales
    int H, block_size;
    long long rows;      // sequences * kv heads
    uint32_t* state;     // in place: [0] the next ticket, [1 + row * chunks + c] reads done
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kMoveThreads = 256, kMoveDeep = 8;

// U: 16-byte units of a K (V) cell; NS: scales; chunk tokens so that a thread has eight units.
template <int U, int NS, bool IN_PLACE>
__global__ __launch_bounds__(kMoveThreads) void compact_kv_kernel(const CompactArgs a) {
    constexpr int T = kMoveThreads * kMoveDeep / (2 * U);
    constexpr int kScales = NS ? T * NS / kMoveThreads : 1;
    static_assert(NS == 0 || T * NS % kMoveThreads == 0, "whole rounds of scales");
    constexpr uint64_t kNone = ~0ull;
    __shared__ uint64_t page[2][T];  // the page's offset, from and to (kNone: not moved)
    __shared__ uint32_t cell[2][T];
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x;
    long long b = (long long)blockIdx.y * gridDim.x + blockIdx.x;
    if constexpr (IN_PLACE) {
        if (tid == 0) ticket = atomicAdd(&a.state[0], 1u);
        __syncthreads();
        b = ticket;
    }
    if (b >= a.rows * a.chunks) return;
    const long long row = b / a.chunks;
    const int c = (int)(b - row * a.chunks), s = (int)(row / a.H), h = (int)(row - (long long)s * a.H);
    const int32_t* __restrict__ kept = a.kept + row * a.budget;
    const int32_t* __restrict__ from = a.tables + (size_t)s * a.max_blocks;
    const int32_t* __restrict__ to = a.out_tables + (size_t)s * a.out_max_blocks;
    for (int k = tid; k < T; k += kMoveThreads) {
        const int j = c * T + k, src = j < a.budget ? kept[j] : -1;
        const int sp = src / a.block_size, dp = j / a.block_size;
        // (in place a token that stays, or one that the order of kept forbids)
        bool move = src >= 0 && sp < a.max_blocks && dp < a.out_max_blocks && (!IN_PLACE || src > j);
        const int si = move ? from[sp] : -1, di = move ? to[dp] : -1;
        move = si >= 0 && di >= 0;
        // (what is not moved is read from the pool's first cell: no load hangs on a condition)
        page[0][k] = move ? (uint64_t)si * a.page_size : 0;
        page[1][k] = move ? (uint64_t)di * a.page_size : kNone;
        cell[0][k] = move ? (uint32_t)((src - sp * a.block_size) * a.H + h) : 0;
        cell[1][k] = (uint32_t)((j - dp * a.block_size) * a.H + h);
    }
    __syncthreads();
    u4 v[kMoveDeep];
    uint16_t sc[kScales];
    const auto unit = [&](int k, int& tok, uint64_t& off) {
        const int x = k * kMoveThreads + tid, part = x / (T * U), y = x - part * (T * U);
        tok = y / U;
        off = a.unit_off[part];
        return y - tok * U;
    };
    const auto scale = [&](int k, int& tok, uint64_t& off) {
        const int x = k * kMoveThreads + tid, part = x / T;
        tok = x - part * T;
        off = a.scale_off[part];
    };
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
        int tok;
        uint64_t off;
        const int u = unit(k, tok, off);
        v[k] = *reinterpret_cast<const u4a2*>(a.pool + page[0][tok] + off + (uint64_t)cell[0][tok] * (16 * U) + u * 16);
    }
    if constexpr (NS > 0) {
#pragma unroll
        for (int k = 0; k < kScales; ++k) {
            int tok;
            uint64_t off;
            scale(k, tok, off);
            sc[k] = ld_u16(a.pool + page[0][tok] + off + (uint64_t)cell[0][tok] * 2);
        }
    }
    if constexpr (IN_PLACE) {
        uint32_t* done = a.state + 1 + row * a.chunks;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's reads have returned
        __syncthreads();
        if (tid == 0) __hip_atomic_store(&done[c], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int k = tid; k < c; k += kMoveThreads)
            while (!__hip_atomic_load(&done[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) __builtin_amdgcn_s_sleep(1);
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
        int tok;
        uint64_t off;
        const int u = unit(k, tok, off);
        if (page[1][tok] != kNone)
            *reinterpret_cast<u4a2*>(a.pool + page[1][tok] + off + (uint64_t)cell[1][tok] * (16 * U) + u * 16) = v[k];
    }
    if constexpr (NS > 0) {
#pragma unroll
        for (int k = 0; k < kScales; ++k) {
            int tok;
            uint64_t off;
            scale(k, tok, off);
            if (page[1][tok] != kNone)
                *reinterpret_cast<uint16_t*>(a.pool + page[1][tok] + off + (uint64_t)cell[1][tok] * 2) = sc[k];
        }
    }
}

__global__ __launch_bounds__(256) void clear_kernel(uint32_t* p, long long n) {
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += (long long)gridDim.x * 256) p[k] = 0;
}

dim3 grid_of(long long blocks) {
    const unsigned x = (unsigned)std::min<long long>(blocks, 1 << 23);
    return dim3(x, (unsigned)((blocks + x - 1) / x));
}

template <int U, int NS>
void launch_move(CompactArgs a, bool in_place, hipStream_t stream) {
    constexpr int T = kMoveThreads * kMoveDeep / (2 * U);
    a.chunks = (a.budget + T - 1) / T;
    const long long blocks = a.rows * a.chunks;
    if (blocks >= (1LL << 31)) throw Error("compact_kv: too many (sequence, kv head, chunk) triples (2^31)");
    if (!in_place) {
        hipLaunchKernelGGL((compact_kv_kernel<U, NS, false>), grid_of(blocks), dim3(kMoveThreads), 0, stream, a);
        check_launch("compact_kv_kernel");
        return;
    }
    const WorkspaceTurn turn(stream);
    a.state = static_cast<uint32_t*>(Scratch{}.get(stream, (1 + (size_t)blocks) * 4, "compact_kv"));
    hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<long long>((blocks + 256) / 256, 1024)), dim3(256), 0, stream,
                       a.state, blocks + 1);
    check_launch("compact_kv_clear_kernel");
    hipLaunchKernelGGL((compact_kv_kernel<U, NS, true>), grid_of(blocks), dim3(kMoveThreads), 0, stream, a);
    check_launch("compact_kv_kernel");
}

bool aligned(uint64_t v, uint64_t a) { return (v & (a - 1)) == 0; }
bool aligned(const void* p, uint64_t a) { return aligned(reinterpret_cast<uintptr_t>(p), a); }

template <class F>
int evict_entry(void* stream, F&& f) {
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

// units: 16-byte units of a K cell; scales: the regions of 16-bit scales.
void compact(const char* name, CompactArgs a, int units, int scales, int D, int num_seqs, bool dense, void* stream) {
    const std::string w = std::string(name) + ": ";
    if (D != 64 && D != 128) throw Error(w + "head_dim must be 64 or 128");
    if (num_seqs < 0) throw Error(w + "num_seqs must be >= 0");
    if (a.budget <= 0) throw Error(w + "budget must be > 0");
    if (a.max_blocks <= 0 || a.out_max_blocks <= 0) throw Error(w + "max_blocks_per_seq must be > 0");
    if ((long long)a.max_blocks * a.block_size > (1LL << 31) - 1 ||
        (long long)a.out_max_blocks * a.block_size > (1LL << 31) - 1 || a.budget > (1 << 30))
        throw Error(w + "a sequence's tokens must fit in 31 bits");
    const uint64_t cells = (uint64_t)a.block_size * a.H;
    const auto outside = [&](uint64_t off, uint64_t size) {
        return off > a.page_size || cells * size > a.page_size - off;
    };
    for (const uint64_t off : a.unit_off)
        if (outside(off, 16 * units)) throw Error(w + "layout does not match cfg (a region ends past the page)");
    for (int k = 0; k < scales; ++k)
        if (outside(a.scale_off[k], 2)) throw Error(w + "layout does not match cfg (a region ends past the page)");
    const uint64_t al = dense ? 16 : 2;
    uint64_t offs = a.page_size | a.unit_off[0] | a.unit_off[1];
    if (!aligned(a.pool, al) || !aligned(offs, al) || !aligned(a.scale_off[0] | a.scale_off[1] | a.scale_off[2], 2))
        throw Error(w + (dense ? "page_pool, page size and offsets must be 16-byte aligned"
                               : "page_pool, page size and offsets must be 2-byte aligned"));
    a.rows = (long long)num_seqs * a.H;
    if (a.rows == 0) return;
    const bool in_place = !a.out_tables;
    if (in_place) {
        a.out_tables = a.tables;
        a.out_max_blocks = a.max_blocks;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (units * 4 + scales) {
        case 16 * 4: return launch_move<16, 0>(a, in_place, st);
        case 8 * 4: return launch_move<8, 0>(a, in_place, st);
        case 4 * 4 + 3: return launch_move<4, 3>(a, in_place, st);
        case 2 * 4 + 3: return launch_move<2, 3>(a, in_place, st);
        case 4 * 4 + 2: return launch_move<4, 2>(a, in_place, st);
        default: return launch_move<2, 2>(a, in_place, st);
    }
}

CompactArgs compact_args(uint8_t* pool, const int32_t* tables, int max_blocks, const int32_t* kept, int budget,
                         const int32_t* out_tables, int out_max_blocks) {
    CompactArgs a{};
    a.pool = pool;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.kept = kept;
    a.budget = budget;
    a.out_tables = out_tables;
    a.out_max_blocks = out_tables ? out_max_blocks : max_blocks;
    return a;
}

void take_geom(CompactArgs& a, const PageGeom& g) {
    a.page_size = g.page_size;
    a.unit_off[0] = g.kc_off;
    a.unit_off[1] = g.vc_off;
    a.H = g.H;
    a.block_size = g.block_size;
}

}  // namespace
}  // namespace tq

extern "C" int tq_launch_select_kv(const float* scores, int64_t score_stride, const int32_t* kv_len, int num_seqs,
                                   int num_kv_heads, int max_kv_len, int budget, int sink, int recent, int32_t* kept,
                                   int32_t* new_len, float* out_scores, int64_t out_stride, void* stream) {
    if (!scores || !kv_len || !kept) return -1;
    return tq::evict_entry(stream, [&] {
        const std::string w = "select_kv: ";
        if (num_seqs < 0 || num_kv_heads <= 0) throw tq::Error(w + "num_seqs must be >= 0 and num_kv_heads > 0");
        if (max_kv_len < 0 || max_kv_len > (1 << 30)) throw tq::Error(w + "max_kv_len must be in [0, 2^30]");
        if (budget <= 0 || budget > (1 << 30)) throw tq::Error(w + "budget must be in [1, 2^30]");
        if (sink < 0 || recent < 0 || (long long)sink + recent > budget)
            throw tq::Error(w + "sink and recent must be >= 0 and together at most budget");
        if (score_stride < max_kv_len || score_stride >= (int64_t(1) << 40))
            throw tq::Error(w + "score_stride must be at least max_kv_len");
        if (out_scores && (out_stride < max_kv_len || out_stride >= (int64_t(1) << 40)))
            throw tq::Error(w + "out_stride must be at least max_kv_len");
        if (out_scores == scores && out_stride != score_stride)
            throw tq::Error(w + "in place, out_stride must be score_stride");
        if (!tq::aligned(scores, 4) || !tq::aligned(out_scores, 4)) throw tq::Error(w + "scores must be 4-byte aligned");
        const long long rows = (long long)num_seqs * num_kv_heads;
        if (rows > (1 << 22) - 1) throw tq::Error(w + "num_seqs * num_kv_heads must be less than 2^22");
        if (rows == 0) return;
        const tq::SelectArgs a{scores,  score_stride, out_stride, kv_len, kept, new_len, out_scores,
                               num_kv_heads, max_kv_len, budget, sink, recent};
        hipLaunchKernelGGL(tq::select_kv_kernel, dim3((unsigned)rows), dim3(tq::kThreads), 0,
                           static_cast<hipStream_t>(stream), a);
        tq::check_launch("select_kv_kernel");
    });
}

extern "C" int tq_launch_dense_compact_kv(uint8_t* page_pool, const int32_t* block_tables, int max_blocks_per_seq,
                                          const int32_t* kept, int budget, const int32_t* out_block_tables,
                                          int out_max_blocks_per_seq, const TQDensePageLayout* layout,
                                          const TQConfig* cfg, int num_seqs, void* stream) {
    if (!page_pool || !block_tables || !kept || !layout || !cfg) return -1;
    return tq::evict_entry(stream, [&] {
        tq::CompactArgs a = tq::compact_args(page_pool, block_tables, max_blocks_per_seq, kept, budget,
                                             out_block_tables, out_max_blocks_per_seq);
        const tq::DenseGeom g = tq::dense_geom(*cfg, *layout);
        a.page_size = g.page_size;
        a.unit_off[0] = g.k_off;
        a.unit_off[1] = g.v_off;
        a.H = g.H;
        a.block_size = g.block_size;
        tq::compact("dense_compact_kv", a, g.D / 8, 0, g.D, num_seqs, true, stream);
    });
}

extern "C" int tq_launch_turbo_prod_compact_kv(uint8_t* page_pool, const int32_t* block_tables,
                                               int max_blocks_per_seq, const int32_t* kept, int budget,
                                               const int32_t* out_block_tables, int out_max_blocks_per_seq,
                                               const TQTurboProdPageLayout* layout, const TQConfig* cfg,
                                               int num_seqs, void* stream) {
    if (!page_pool || !block_tables || !kept || !layout || !cfg) return -1;
    return tq::evict_entry(stream, [&] {
        tq::CompactArgs a = tq::compact_args(page_pool, block_tables, max_blocks_per_seq, kept, budget,
                                             out_block_tables, out_max_blocks_per_seq);
        const tq::PageGeom g = tq::prod_geom(*cfg, *layout);
        tq::take_geom(a, g);
        a.scale_off[0] = g.kres_off;
        a.scale_off[1] = g.ks_off;
        a.scale_off[2] = g.vs_off;
        tq::compact("turbo_prod_compact_kv", a, g.D / 32, 3, g.D, num_seqs, false, stream);
    });
}

extern "C" int tq_launch_turbo_mse_compact_kv(uint8_t* page_pool, const int32_t* block_tables,
                                              int max_blocks_per_seq, const int32_t* kept, int budget,
                                              const int32_t* out_block_tables, int out_max_blocks_per_seq,
                                              const TQTurbomsePageLayout* layout, const TQConfig* cfg,
                                              int num_seqs, void* stream) {
    if (!page_pool || !block_tables || !kept || !layout || !cfg) return -1;
    return tq::evict_entry(stream, [&] {
        tq::CompactArgs a = tq::compact_args(page_pool, block_tables, max_blocks_per_seq, kept, budget,
                                             out_block_tables, out_max_blocks_per_seq);
        const tq::PageGeom g = tq::mse_geom(*cfg, *layout);
        tq::take_geom(a, g);
        a.scale_off[0] = g.ks_off;
        a.scale_off[1] = g.vs_off;
        tq::compact("turbo_mse_compact_kv", a, g.D / 32, 2, g.D, num_seqs, false, stream);
    });
}
