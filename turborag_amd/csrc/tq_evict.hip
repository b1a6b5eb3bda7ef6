// tq_evict.hip — eviction from paged caches: the tokens that a budget keeps, by their
// scores, and the move of their cells to the front.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "tq_device.h"

namespace tq {
namespace {

using namespace dev;

// ---------------------------------------------------------------------------
// Selection.  One workgroup per (sequence, kv head): a radix search of the lowest kept
// score over the bits of an order-preserving key, digits of 10, 11 and 11 bits counted
// in LDS, which ends as soon as all tokens of the digit are kept; then the kept tokens
// in order, from a bit per token in LDS, whose words' counts are summed up over the
// threads.  A lane has kDeep tokens in registers, a tile of the workgroup; a row of one
// tile is read once for its keys.
// 4 bytes a token: bound by the latency of the steps, one after the other, in one compute
// unit a row (64 rows to 32K tokens 19.8 us, of ~35,000 cycles the load 8, the first digit 7,
// the others 5 to 10, the marks 3 and the scores' gather 6 thousand; 1,143 tokens 7.2 us).
// The gather from a list in LDS instead of kept: no gain (19.9).
// ---------------------------------------------------------------------------
struct SelectArgs {
    const float* scores;
    int64_t stride, out_stride;  // from one head's scores to the next
    const int32_t* kv_len;
    int32_t *kept, *new_len;  // new_len or null
    float* out;               // null, or the kept tokens' scores; may be the scores
    int heads, max_kv, budget, sink, recent;
};

// Larger scores have larger keys; -0 is 0, NaN is below everything.  Keys lie between
// those of tokens that are none (0) and of tokens that stay whatever their score (~0).
constexpr uint32_t kNoToken = 0u, kStays = ~0u;
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);
    return f != f ? 1u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

// f(0), f(1), ..., as constants.
template <int N, int K = 0, class F>
__device__ __forceinline__ void for_each_lane(F&& f) {
    if constexpr (K < N) {
        f(std::integral_constant<int, K>{});
        for_each_lane<N, K + 1>(f);
    }
}
// The wave's mask m into lane K of `to`.  (The wait states between a vector instruction's
// scalar result and the next one that reads it, which the compiler does not see here.)
template <int K>
__device__ __forceinline__ void into_lane(uint2& to, uint64_t m) {
    asm("s_nop 3\n\tv_writelane_b32 %0, %2, %4\n\tv_writelane_b32 %1, %3, %4"
        : "+v"(to.x), "+v"(to.y)
        : "s"((uint32_t)m), "s"((uint32_t)(m >> 32)), "n"(K));
}

// The first digit's counters lie in COPIES side by side, a lane's by its number: scores of
// a softmax have few exponents, and lanes that count at one address or bank take turns.
template <int WAVES, int COPIES, int kDeep>
__global__ __launch_bounds__(64 * WAVES) void select_kv_kernel(const SelectArgs a) {
    constexpr int kThreads = 64 * WAVES, kTile = kThreads * kDeep;
    static_assert(COPIES >= 4 && 1024 * COPIES >= 2048, "counters");
    __shared__ __attribute__((aligned(16))) uint32_t bins[1024 * COPIES];
    __shared__ uint32_t above[WAVES], found[3];
    __shared__ uint2 marks[2][kTile / 64];  // kept for certain; with the lowest kept key
    __shared__ int2 counts[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x;
    const int s = (int)(row / a.heads), B = a.budget;
    const int L = min(max(a.kv_len[s], 0), a.max_kv), n = min(L, B);
    const float* x = a.scores + row * a.stride;
    int32_t* kept = a.kept + row * B;
    float* out = a.out ? a.out + row * a.out_stride : nullptr;
    if (a.new_len && row == (int64_t)s * a.heads && tid == 0) a.new_len[s] = n;

    if (L <= B) {
        for (int j = tid; j < B; j += kThreads) kept[j] = j < L ? j : -1;
        if (out && out != x)
            for (int j = tid; j < L; j += kThreads) out[j] = x[j];
        if (out)
            for (int j = n + tid; j < a.max_kv; j += kThreads) out[j] = 0.0f;
        return;
    }
    const auto clear_rest = [&] {  // (four at a time; the row may begin at any float)
        typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
        for (int j = n + 4 * tid; j < a.max_kv; j += 4 * kThreads) {
            if (j + 4 <= a.max_kv)
                *reinterpret_cast<f4u*>(out + j) = f4u{0.0f, 0.0f, 0.0f, 0.0f};
            else
                for (int k = j; k < a.max_kv; ++k) out[k] = 0.0f;
        }
    };
    const bool in_place = out == x;
    if (out && !in_place) clear_rest();
    // [lo, hi): the tokens that their scores decide on.
    const int lo = a.sink, hi = L - a.recent, tiles = (L + kTile - 1) / kTile;
    constexpr int per = 64 * kDeep;  // a wave's tokens of a tile, in a row, lane by lane
    uint32_t keys[kDeep];
    const auto load = [&](int tile) __attribute__((always_inline)) {
        const int t0 = tile * kTile + wv * per + lane, end = min(tile * kTile + (wv + 1) * per, L);
#pragma unroll
        for (int k = 0; k < kDeep; ++k) keys[k] = __float_as_uint(x[min(t0 + k * 64, L - 1)]);
        const int w0 = tile * kTile + wv * per;  // (the same in every lane)
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            keys[k] = key_of(__uint_as_float(keys[k]));
            if (w0 + k * 64 < lo || w0 + k * 64 + 64 > min(hi, end)) {
                const int t = t0 + k * 64;
                keys[k] = t >= end ? kNoToken : t < lo || t >= hi ? kStays : keys[k];
            }
        }
    };
    // f(key, k) of the wave's tokens of the tile.
    const auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kDeep; ++k) f(keys[k], k);
    };
    load(0);

    uint32_t want = (uint32_t)(B - a.sink - a.recent), prefix = 0;
    int shift = 32;
    bool ties = false;  // of the tokens with the prefix only the first `want` are kept
    const auto digit = [&](auto first, auto width) __attribute__((always_inline)) {
        constexpr bool kFirst = decltype(first)::value;
        constexpr int kBits = decltype(width)::value, kBins = 1 << kBits, kMine = kBins / kThreads;
        constexpr int kCopies = kFirst ? COPIES : 1;
        const int from = shift;
        shift -= kBits;
        for (int k = tid * 4; k < kBins * kCopies; k += kThreads * 4)
            *reinterpret_cast<uint4*>(bins + k) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        // The first digit counts every lane's keys: kStays alone has the highest one (an
        // infinity's is one less), and kNoToken's are subtracted from the lowest.  Later, none
        // but counted keys have the prefix, unless it is 0.
        const bool checked = prefix == 0;
        for (int tile = 0; tile < tiles; ++tile) {
            if (tiles > 1 && (!kFirst || tile)) load(tile);
            each([&](uint32_t key, int) {
                if (kFirst || (key >> (from & 31) == prefix && (!checked || key != kNoToken)))
                    atomicAdd(&bins[(key >> shift & (kBins - 1)) * kCopies + (lane & (kCopies - 1))], 1u);
            });
        }
        __syncthreads();
        // The digit at which the tokens from the top reach `want`: kMine bins a thread,
        // from the top down.
        uint32_t mine[kMine], sum = 0;
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            const int d = kBins - 1 - (tid * kMine + e);
            if constexpr (kFirst) {
                mine[e] = 0;
#pragma unroll
                for (int k = 0; k < COPIES; k += 4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(bins + d * COPIES + ((k + 4 * tid) & (COPIES - 1)));
                    mine[e] += w.x + w.y + w.z + w.w;
                }
                if (d == kBins - 1) mine[e] = 0;
                if (d == 0) mine[e] -= (uint32_t)(tiles * kTile - L);
            } else {
                mine[e] = bins[d];
            }
            sum += mine[e];
        }
        uint32_t up = sum;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(up, m, 64);
            if (lane >= m) up += o;
        }
        if (lane == 63) above[wv] = up;
        __syncthreads();
        uint32_t before = up - sum;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) before += w < wv ? above[w] : 0u;
        if (before < want && before + sum >= want) {
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                if (before < want && before + mine[e] >= want) {
                    found[0] = (uint32_t)(kBins - 1 - (tid * kMine + e));
                    found[1] = want - before;
                    found[2] = mine[e];
                }
                before += mine[e];
            }
        }
        __syncthreads();
        prefix = prefix << kBits | found[0];
        want = found[1];
        ties = found[2] != want;
        if (ties) __syncthreads();  // (found is written again)
    };
    if (want) {
        digit(std::true_type{}, std::integral_constant<int, 10>{});
        for (int k = 0; k < 2 && ties; ++k) digit(std::false_type{}, std::integral_constant<int, 11>{});
    }
    // Kept: keys from `sure` on and, of those from `tie` on, the first `want`.
    const bool none = a.sink + a.recent == B;
    const uint32_t tie = none ? kStays : max(prefix << shift, 1u);
    const uint32_t sure = none ? kStays : ties ? (prefix + 1u) << shift : tie;
    int at = 0, equal = 0;  // kept tokens and equal ones of the tiles so far
    for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1) load(tile);
        uint2 certain = {0, 0}, same = {0, 0};  // lane k: the bits of the wave's tokens 64 k ..
        for_each_lane<kDeep>([&](auto k) { into_lane<k.value>(certain, __ballot(keys[k.value] >= sure)); });
        if (sure != tie)
            for_each_lane<kDeep>(
                [&](auto k) { into_lane<k.value>(same, __ballot(keys[k.value] - tie < sure - tie)); });
        if (lane < kDeep) {
            marks[0][wv * kDeep + lane] = certain;
            marks[1][wv * kDeep + lane] = same;
        }
        __syncthreads();
        // A thread has 32 tokens of the tile, which lie in a row.
        constexpr int kWords = kTile / 32;
        static_assert(kWords <= kThreads, "a word per thread");
        uint32_t keep = 0, ties_of = 0;
        if (tid < kWords) {
            keep = reinterpret_cast<const uint32_t*>(marks[0])[tid];
            ties_of = reinterpret_cast<const uint32_t*>(marks[1])[tid];
        }
        int2 up = make_int2(__popc(keep), __popc(ties_of));
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int ox = __shfl_up(up.x, m, 64), oy = __shfl_up(up.y, m, 64);
            if (lane >= m) up.x += ox, up.y += oy;
        }
        if (lane == 63) counts[wv] = up;
        __syncthreads();
        int base = at + up.x - __popc(keep), eq = equal + up.y - __popc(ties_of), next = at, next_eq = equal;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int2 e = counts[w];
            base += w < wv ? e.x : 0;
            eq += w < wv ? e.y : 0;
            next += e.x;
            next_eq += e.y;
        }
        const int quota = (int)want;  // of the equal ones
        base += min(eq, quota) - min(equal, quota);
        while (ties_of && eq < quota) {
            keep |= ties_of & -ties_of;
            ties_of &= ties_of - 1;
            ++eq;
        }
        const int t0 = tile * kTile + tid * 32;
        while (keep) {
            kept[base++] = t0 + __ffs(keep) - 1;
            keep &= keep - 1;
        }
        at = next + min(next_eq, quota) - min(equal, quota);
        equal = next_eq;
        if (tiles > 1) __syncthreads();  // (marks and counts are written again)
    }
    if (out) {
        // In order: place j takes the score of a token at j or behind it, so in place none is
        // overwritten before it is read.
        __threadfence_block();
        __syncthreads();
        constexpr int kPlaces = 4;
        for (int j0 = 0; j0 < n; j0 += kPlaces * kThreads) {
            float f[kPlaces];
#pragma unroll
            for (int k = 0; k < kPlaces; ++k) f[k] = x[kept[min(j0 + k * kThreads + tid, n - 1)]];
            if (in_place) __syncthreads();
#pragma unroll
            for (int k = 0; k < kPlaces; ++k) {
                const int j = j0 + k * kThreads + tid;
                if (j < n) out[j] = f[k];
            }
            if (in_place) __syncthreads();
        }
        if (in_place) clear_rest();
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
// reads are done, and waits with its writes for those before it that keep a token from
// within [a, b) (kept rises: between their first and last one).  A (sequence, kv
// head)'s chunks are taken by tickets in that order, so what a workgroup waits for has
// begun, and reads wait for nothing: every wait ends.  (Dense, 32
// sequences to 4,096 tokens in place: 92.7 us with one counter for all, 81.9 with one each,
// 78.9 without the waits that are not needed.  The kernel alone 72, into other pages 56;
// turbo_prod 30 and 26: what is left is read, then waited for, then written in turn.)
// ---------------------------------------------------------------------------
struct CompactArgs {
    uint8_t* pool;
    const int32_t *tables, *out_tables, *kept;
    int max_blocks, out_max_blocks, budget, chunks;
    uint64_t page_size;
    uint64_t unit_off[2], scale_off[3];  // K, V; scales
    int H, block_size;
    long long rows;      // sequences * kv heads
    uint32_t* state;     // in place: [row] its next ticket, [rows + row * chunks + c] reads done
    uint32_t* lost;      // in place: host memory, set where chunks stay unwritten; or null
    int polls;           // in place: of a wait, at most
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kMoveThreads = 256, kMoveDeep = 8;
// Waits of some microseconds are given up after about a second, which takes two graphs of one
// stream replayed at once, against the rule: both end, no cell that is still to be read is
// written over, and the next call says that cells were not moved.
constexpr int kMostPolls = 1 << 20;

// Cells of whole cache lines go past the caches (dense, 32 sequences to 4,096 tokens each,
// 258 MB: 58.6 -> 54.4 us; 8 kv heads 60.2 -> 56.4); parts of lines are put together there
// (turbo_prod 21.5 against 24.9).
template <int U>
__device__ __forceinline__ void store_unit(uint8_t* p, u4 v) {
    if constexpr (U >= 8)
        __builtin_nontemporal_store((u4a2)v, reinterpret_cast<u4a2*>(p));
    else
        *reinterpret_cast<u4a2*>(p) = v;
}

__device__ __forceinline__ void say_lost(const CompactArgs& a) {
    if (a.lost) __hip_atomic_store(a.lost, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// U: 16-byte units of a K (V) cell; NS: scales; chunk tokens so that a thread has eight units.
template <int U, int NS, bool IN_PLACE>
__global__ __launch_bounds__(kMoveThreads) void compact_kv_kernel(const CompactArgs a) {
    constexpr int T = kMoveThreads * kMoveDeep / (2 * U);
    constexpr int kScales = NS ? T * NS / kMoveThreads : 1;
    static_assert(NS == 0 || T * NS % kMoveThreads == 0, "whole rounds of scales");
    constexpr uint64_t kNone = ~0ull;
    __shared__ uint64_t page[2][T];  // the page's offset, from and to (kNone: not moved)
    __shared__ uint32_t cell[2][T];
    __shared__ uint32_t ticket, gave_up;
    const int tid = threadIdx.x;
    const long long b = (long long)blockIdx.y * gridDim.x + blockIdx.x;
    if (b >= a.rows * a.chunks) return;
    const long long row = b / a.chunks;
    int c = (int)(b - row * a.chunks);
    if constexpr (IN_PLACE) {
        if (tid == 0) {
            ticket = atomicAdd(&a.state[row], 1u);
            gave_up = 0;
        }
        __syncthreads();
        // (state that another call's kernels share may hold any bits: nothing out of bounds)
        if (ticket >= (uint32_t)a.chunks) {
            if (tid == 0) say_lost(a);
            return;
        }
        c = (int)ticket;
    }
    const int s = (int)(row / a.H), h = (int)(row - (long long)s * a.H);
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
        uint32_t* done = a.state + a.rows + row * a.chunks;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's reads have returned
        __syncthreads();
        if (tid == 0) __hip_atomic_store(&done[c], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int k = tid; k < c; k += kMoveThreads)  // (unsigned: a hole in kept counts as any token)
            if (kept[k * T] < (c + 1) * T && (uint32_t)kept[k * T + T - 1] >= (uint32_t)(c * T)) {
                int polls = 0;
                for (; polls < a.polls; ++polls) {
                    if (__hip_atomic_load(&done[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) break;
                    __builtin_amdgcn_s_sleep(1);
                }
                if (polls >= a.polls) gave_up = 1;
            }
        __syncthreads();
        if (gave_up) {
            if (tid == 0) say_lost(a);
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
        int tok;
        uint64_t off;
        const int u = unit(k, tok, off);
        if (page[1][tok] != kNone)
            store_unit<U>(a.pool + page[1][tok] + off + (uint64_t)cell[1][tok] * (16 * U) + u * 16, v[k]);
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

// The tickets (the first `rows` words) and the flags behind them.
__global__ __launch_bounds__(256) void clear_kernel(uint32_t* p, long long n, long long rows, uint32_t first) {
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += (long long)gridDim.x * 256)
        p[k] = k < rows ? first : 0;
}

// What tests set (tq_test_compact).
std::atomic<uint32_t> g_first_ticket{0};
std::atomic<int> g_polls{kMostPolls};

// A word of host memory for all calls, which kernels write if they leave cells unmoved.  Never
// freed: graphs hold it.  (Also made within a capture, which nothing that is not recorded ends
// in the relaxed mode; none to be had: nothing is said.)
std::atomic<uint32_t*> g_lost{nullptr};
uint32_t* lost_word() {
    uint32_t* p = g_lost.load(std::memory_order_acquire);
    if (p) return p;
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    if ((p = g_lost.load(std::memory_order_acquire))) return p;
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    void* mem = nullptr;
    if (hipHostMalloc(&mem, sizeof(uint32_t), hipHostMallocPortable | hipHostMallocMapped) != hipSuccess) mem = nullptr;
    if (relaxed) (void)hipThreadExchangeStreamCaptureMode(&mode);
    if (!mem) {
        (void)hipGetLastError();
        return nullptr;
    }
    p = static_cast<uint32_t*>(mem);
    *p = 0;
    g_lost.store(p, std::memory_order_release);
    return p;
}
// Once for all that were lost before.
void report_lost() {
    uint32_t* p = g_lost.load(std::memory_order_acquire);
    if (p && __atomic_load_n(p, __ATOMIC_RELAXED) && __atomic_exchange_n(p, 0u, __ATOMIC_RELAXED))
        throw Error("compact_kv: an earlier in-place call left cells unmoved, because another call's kernels wrote over "
                    "its workspace (graphs of one stream replayed at once?); this call did nothing");
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
    const long long words = a.rows + blocks;
    a.lost = lost_word();
    a.polls = g_polls.load(std::memory_order_relaxed);
    a.state = static_cast<uint32_t*>(Scratch{}.get(stream, (size_t)words * 4, "compact_kv"));
    hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<long long>((words + 255) / 256, 1024)), dim3(256), 0, stream,
                       a.state, words, a.rows, g_first_ticket.load(std::memory_order_relaxed));
    check_launch("compact_kv_clear_kernel");
    hipLaunchKernelGGL((compact_kv_kernel<U, NS, true>), grid_of(blocks), dim3(kMoveThreads), 0, stream, a);
    check_launch("compact_kv_kernel");
}

bool aligned(uint64_t v, uint64_t a) { return (v & (a - 1)) == 0; }
bool aligned(const void* p, uint64_t a) { return aligned(reinterpret_cast<uintptr_t>(p), a); }

template <class F>
int evict_entry(void* stream, F&& f) {
    try {
        report_lost();
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

// For tests: the first ticket of in-place moves (0, but for a workspace that another call's
// kernels have written over), and the polls after which a wait is given up (< 0: as ever).
extern "C" __attribute__((visibility("default"))) int tq_test_compact(uint32_t first_ticket, int polls) {
    tq::g_first_ticket.store(first_ticket);
    tq::g_polls.store(polls < 0 ? tq::kMostPolls : polls);
    return 0;
}

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
        const hipStream_t st = static_cast<hipStream_t>(stream);
        if (max_kv_len <= 2048)
            hipLaunchKernelGGL((tq::select_kv_kernel<4, 8, 8>), dim3((unsigned)rows), dim3(256), 0, st, a);
        else if (max_kv_len <= 8192)
            hipLaunchKernelGGL((tq::select_kv_kernel<16, 32, 8>), dim3((unsigned)rows), dim3(1024), 0, st, a);
        else
            hipLaunchKernelGGL((tq::select_kv_kernel<16, 32, 32>), dim3((unsigned)rows), dim3(1024), 0, st, a);
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
