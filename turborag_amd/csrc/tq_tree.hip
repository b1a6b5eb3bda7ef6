// tq_tree.hip — attention of drafted token trees over paged caches: dense
// pages (fp16, bf16), turbo_prod and turbo_mse pages.
//
// Row (token r of sequence s, query head) attends the tokens t of s with
// t < prefix_len[s], or t = prefix_len[s] + j with bit j of the row's mask:
//   out = sum_t softmax_t(<q, k_t> / sqrt(D)) v_t.
// Compressed pages hold k and v rotated (an orthogonal transform), so q is
// rotated the same way, and the output rotated back.
//
// One pass over a sequence's tokens for up to 256 query rows (drafted tokens x
// query heads of a kv head), with a running reference and sum per row; the
// sequences' tokens are one line of work cut into equal parts, one per
// workgroup, and what was cut is merged by a second launch.  Measured (MI355X,
// 16 query heads on 2 kv heads, head_dim 128; kernels alone):
//  - dense bf16, 32 sequences of 1,024 to 32,768 tokens, 4 to 8 drafted tokens
//    each, 556 MB: a call 118 us, 4.7 TB/s where a copy of 1 GiB runs at 5.2: bound
//    by HBM;
//  - dense fp16, 64 drafted tokens over 32,768: 46 + 9 us, 375 TFLOP/s of the split
//    (an 8,192^3 product of the library's: 1,300).  Of a workgroup's 77,000 cycles
//    6,800 are for each of nine chunks (two waves per SIMD: ~3,100 of matrix
//    instructions, the rest the softmax's vector instructions), 9,500 for the chain
//    lengths -> page ids -> rows, 4,500 for the partial sums, 33 MB in all;
//  - the same over turbo_prod: 65 + 9 us, 10,900 cycles a chunk: more matrix
//    instructions (K and q as fp16 pairs), LDS cycles, and the decode (~100 vector
//    instructions per wave and chunk);
//  - turbo_prod, 32 sequences of 300 to 8,192 tokens: 46 + 8 us, the same;
//  - one sequence of 1,143 tokens, 5 drafted: 7.2 + 4.2 us, latency: lengths -> page
//    ids -> rows -> products -> partial sums, then the merge's launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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
    int max_blocks, mask_words, hq, group, seqs, tokens, max_kv;  // group: query heads per kv head
};

// Base-2 exponent and logarithm as the hardware computes them (~1 ulp).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u4 lds_u4;
typedef __attribute__((address_space(3))) s4 lds_s4;

// C += A B, A [16 x 32] by rows, B [32 x 16] by columns: lane l holds row
// (column) l % 16, k = 8 (l / 16) + 0..7; of C column l % 16, rows
// 4 (l / 16) + 0..3.
template <bool BF>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                       __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Two fp32 -> packed fp16 or bf16, to nearest even, a in the low half.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF) {
        typedef float f2v __attribute__((ext_vector_type(2)));
        typedef __bf16 b2v __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){a, b}, b2v));
    } else {
        typedef float f2v __attribute__((ext_vector_type(2)));
        typedef _Float16 h2v __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){a, b}, h2v));
    }
}

// What pack2's result hi leaves of a and b, packed likewise.
template <bool BF>
__device__ __forceinline__ uint32_t pack2_rest(uint32_t hi, float a, float b) {
    if constexpr (BF) {
        return pack2<BF>(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
    } else {
        uint32_t lo;
        asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\t"
            "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=&v"(lo)
            : "v"(hi), "v"(a), "v"(b));
        return lo;
    }
}

// All ones in the halves of x that are infinite or NaN.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    return ((x & E) == E ? 0xffffu : 0u) | ((x >> 16 & E) == E ? 0xffff0000u : 0u);
}
// 1.0 in the halves of x that are NaN or infinite with sign `neg`.
template <bool BF>
__device__ __forceinline__ uint32_t infinite_ones(uint32_t x, uint32_t neg) {
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u, one = BF ? 0x3f80u : 0x3c00u;
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 32; k += 16) {
        const uint32_t v = x >> k & 0xffffu, m = v & 0x7fffu;
        r |= (m > E || (m == E && v >> 15 == neg)) ? one << k : 0u;
    }
    return r;
}

// One butterfly stage with lane ^ M (16 or 32) of two values: the swap brings a
// value's two halves under each other, and back.
template <int M>
__device__ __forceinline__ void butterfly2(float& a, float& b) {
    const auto swap = [](float u, float w) {
        if constexpr (M == 16)
            return __builtin_amdgcn_permlane16_swap(__float_as_uint(u), __float_as_uint(w), false, false);
        else
            return __builtin_amdgcn_permlane32_swap(__float_as_uint(u), __float_as_uint(w), false, false);
    };
    const auto x = swap(a, b);
    const float u = __uint_as_float(x[0]), w = __uint_as_float(x[1]);
    const auto y = swap(u + w, u - w);
    a = __uint_as_float(y[0]);
    b = __uint_as_float(y[1]);
}
template <int M>
__device__ __forceinline__ float butterfly(float v, int lane) {
    const float o = lane_xor<M>(v);
    return (lane & M) ? o - v : v + o;
}

// ---------------------------------------------------------------------------
// Work of a launch.  An item is one (kv head, sequence, tile of M query rows),
// its chunks of C tokens.  Items lie one behind the other (by head, sequence,
// tile), and workgroup w takes the chunks [w per, (w + 1) per) of that line:
// the same work for every workgroup, whatever the lengths, which only the
// device knows.  A piece is a workgroup's part of an item; only its first and
// its last piece can be cut.  Every item begins with kLead chunks of no tokens:
// beginning a piece costs about as much as they do, so a workgroup with an item's
// beginning inside gets as many chunks less (32 ragged sequences, turbo_prod:
// the last workgroup had ended 10 us after the median one).
// ---------------------------------------------------------------------------
constexpr int kLead = 2;
struct Tiling {
    int m_log, c_log;  // log2 of M, C
    int groups;        // workgroups of the split launch
};
struct Plan {
    int total;  // chunks of one head's items
    int per;    // chunks of a workgroup
};
// One sequence per lane, from sequence `first` on.
struct SeqBlock {
    int first;
    int row0, rows, L, end;  // first token row, drafted tokens, prefix length, kv end
    int chunks, tiles;  // (chunks of an item, kLead among them)
    int before;  // chunks of the head's items before this sequence
};

__device__ __forceinline__ SeqBlock read_seqs(const TreeArgs& a, const Tiling& g, int first, int lane) {
    SeqBlock b;
    b.first = first;
    const int s = min(first + lane, a.seqs - 1);
    const int r0 = a.row_start[s], r1 = a.row_start[s + 1], L = a.prefix[s];
    b.row0 = min(max(r0, 0), a.tokens);
    b.rows = first + lane < a.seqs ? max(min(r1, a.tokens) - b.row0, 0) : 0;
    b.L = max(L, 0);
    b.end = (int)min((long long)b.L + b.rows, (long long)a.max_kv);
    b.chunks = max((b.end + (1 << g.c_log) - 1) >> g.c_log, 1) + kLead;
    b.tiles = (b.rows * a.group + (1 << g.m_log) - 1) >> g.m_log;
    b.before = 0;
    return b;
}
// Sums over the lanes up to this one: within rows of 16 by shifts, then the
// rows' last lanes broadcast to the rows behind (every lane active).
__device__ __forceinline__ int sum_up(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2, 3
    return v;
}
__device__ __forceinline__ SeqBlock load_seqs(const TreeArgs& a, const Tiling& g, int first,
                                              int before, int lane, int& after) {
    SeqBlock b = read_seqs(a, g, first, lane);
    const int cost = b.tiles * b.chunks, up = sum_up(cost);
    b.before = before + up - cost;
    after = before + __builtin_amdgcn_readlane(up, 63);
    return b;
}
// More than 64 sequences: lane k's chunks of the blocks of 64 from k span to
// (k + 1) span, so that a place is found from one sum over lanes and at most
// span blocks.  Returns the chunks of all.
__device__ __forceinline__ int span_of(int seqs) { return (seqs + 4095) / 4096; }
__device__ __forceinline__ int block_sums(const TreeArgs& a, const Tiling& g, int lane, int& mine) {
    const int span = span_of(a.seqs);
    int total = 0;
    mine = 0;
    for (int f = 0; f < a.seqs; f += 256) {  // (four blocks' loads at a time)
        int cost[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const SeqBlock b = read_seqs(a, g, f + k * 64, lane);
            cost[k] = b.tiles * b.chunks;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int sum = __builtin_amdgcn_readlane(sum_up(cost[k]), 63);
            if ((f / 64 + k) / span == lane) mine += sum;
            total += sum;
        }
    }
    return total;
}

__device__ __forceinline__ Plan make_plan(const TreeArgs& a, const Tiling& g, int total) {
    Plan p;
    p.total = total;
    const long long all = (long long)total * a.g.H;
    p.per = max((int)((all + g.groups - 1) / g.groups), 1);
    return p;
}

// A piece, the same in every lane.
struct Piece {
    int h, s, row0, rows, L, end;
    int tile, chunk, chunks;  // place in the item (from kLead on: chunks of tokens); its chunks
};
__device__ __forceinline__ Piece locate(const TreeArgs& a, const Tiling& g, const Plan& p, int at,
                                        int lane, int mine, SeqBlock& b) {
    Piece o;
    o.h = at / p.total;
    const int x = at - o.h * p.total;
    if (a.seqs > 64) {
        int after = __builtin_amdgcn_readlane(b.before + b.tiles * b.chunks, 63);
        if (b.first < 0 || x < __builtin_amdgcn_readlane(b.before, 0) || x >= after) {
            const int step = 64 * span_of(a.seqs), from = sum_up(mine) - mine;
            const int k = max(__popcll(__ballot(from <= x && lane * step < a.seqs)) - 1, 0);
            b = load_seqs(a, g, k * step, __builtin_amdgcn_readlane(from, k), lane, after);
            while (x >= after && b.first + 64 < a.seqs) b = load_seqs(a, g, b.first + 64, after, lane, after);
        }
    }
    // The last sequence that begins at or before x: one without work begins
    // where its successor does, so it is the last only if x is past all work.
    const int k = max(__popcll(__ballot(b.before <= x && b.first + lane < a.seqs)) - 1, 0);
    o.s = b.first + k;
    o.row0 = __builtin_amdgcn_readlane(b.row0, k);
    o.rows = __builtin_amdgcn_readlane(b.rows, k);
    o.L = __builtin_amdgcn_readlane(b.L, k);
    o.end = __builtin_amdgcn_readlane(b.end, k);
    o.chunks = __builtin_amdgcn_readlane(b.chunks, k);
    const int y = x - __builtin_amdgcn_readlane(b.before, k);
    o.tile = y / o.chunks;
    o.chunk = y - o.tile * o.chunks;
    return o;
}

// ---------------------------------------------------------------------------
// The split kernel: NW waves, WR of them side by side over the tile's rows
// (16 RT each), NW / WR over a chunk's tokens (T each).  Both products run
// transposed: S' = K Q' has a query row per lane column and four tokens in a
// lane's registers, so a row's softmax is in-lane but for two lane swaps, and
// the registers are the B operand of O' = V' P' as they are (the k-order of a
// 32-token step is 4 (l / 16) + 0..3 of either 16 tokens; V' is read from its
// token rows in that order by transposing LDS loads).
//
// Weights enter their product with V in two parts of the pages' 16-bit type (fp16
// for compressed pages): ~22 bits (bf16: 16) as in the other attention kernels.
// One part alone, rounded as far as the output is, left flat rows 1.4 times the
// error of fp32 weights; the second costs 64 drafted tokens over 32,768 43.1 ->
// 49.5 us (fp16), 61.4 -> 64.4 (turbo_prod), 32 sequences 115.8 -> 118.2 (bf16), 46.7
// -> 48.9 (turbo_prod).  Logits, sums and references are fp32.  RT = 2: a K or V operand read from LDS serves two
// products; one row tile per wave reads as many bytes as LDS gives.
// ---------------------------------------------------------------------------
template <int FMT, int D, int RT, int WR, int NW>
struct Shape {
    static constexpr bool kTurned = FMT == kProd || FMT == kMse, BF = FMT == kBf16;
    static constexpr int WT = NW / WR;
    // Workgroups of a CU (registers and LDS hold so many).
    static constexpr int kPerCu = kTurned && RT == 1 && WR == 4 ? 3 : WR == 1 && D == 128 ? 1 : 8 / NW;
    static constexpr int T = WR >= 4 ? 64 : 32, C = T * WT, M = 16 * RT * WR;
    static constexpr int kRow = 2 * D, kTile = C * kRow;
    // Buffers of a chunk's tiles (K, V; compressed pages K hi, K lo, V, one buffer
    // where other workgroups of the CU work while it is filled).
    static constexpr int kBufs = kTurned && WR < 8 ? 1 : 2, kTiles = kTurned ? 3 : 2;
    static constexpr int kMerge = WT > 1 ? WT * M * D * 4 : 0;
    static constexpr int kLds = kBufs * kTiles * kTile > kMerge ? kBufs * kTiles * kTile : kMerge;
    // Bytes of codes that a lane decodes at a time, how many of them, lanes per token.
    static constexpr int kLane = T * (D / 2) / (WR * 64), kUnit = kLane < 16 ? kLane : 16;
    static constexpr int KU = kLane / kUnit, kParts = D / 2 / kUnit;
};

constexpr float kAlphaV = 1.5982153f;  // alpha V4[c] is fp16-exact to 9.2e-5 for every c

// 16 bytes per lane from p straight into LDS at byte `lds` (the same in every
// lane) + 16 lane.  In asm, because the compiler waits for loads of its own kind
// before any LDS read that follows; wait_vmem() is the wait.
__device__ __forceinline__ void load_to_lds(const uint8_t* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                     __builtin_amdgcn_readfirstlane(lds)),
                 "v"(p)
                 : "m0", "memory");
}
__device__ __forceinline__ void wait_vmem() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

struct DecodeTables {
    uint32_t v[256];  // code byte -> fp16 pair of alpha V4 (low nibble first)
    // turbo_mse: fp16 pairs of V4, hi and lo; turbo_prod: fp32 pair of K3, the
    // last bit 1 where the residual is subtracted.
    uint2 k[256];
};
// Two table entries of turbo_prod's K and the row's residual RMS -> their
// values level +- re as fp16 pairs, hi and lo = fp16(value - hi).
__device__ __forceinline__ uint2 split_k3(uint2 e, float re) {
    uint32_t s0, s1;  // 1.0, negative where the last bit is 1
    asm("v_lshl_or_b32 %0, %1, 31, 1.0" : "=v"(s0) : "v"(e.x));
    asm("v_lshl_or_b32 %0, %1, 31, 1.0" : "=v"(s1) : "v"(e.y));
    const float x = fmaf(__uint_as_float(s0), re, __uint_as_float(e.x));
    const float y = fmaf(__uint_as_float(s1), re, __uint_as_float(e.y));
    const uint32_t hi = pack2<false>(x, y);
    return make_uint2(hi, pack2_rest<false>(hi, x, y));
}

struct alignas(16) TokenScales {
    float k[128], v[128], lv[128];  // of a chunk's tokens; lv = max(log2 |v|, -25)
};
struct Nothing {};

template <int FMT, int D, int RT, int WR, int NW>
__global__ __launch_bounds__(64 * NW, ((Shape<FMT, D, RT, WR, NW>::kPerCu * NW + 3) / 4))
void tree_split_kernel(const TreeArgs a, const Tiling tl, float* __restrict__ ws, float scale, float inv) {
    using S = Shape<FMT, D, RT, WR, NW>;
    constexpr bool BF = S::BF, kTurned = S::kTurned;
    constexpr int T = S::T, C = S::C, M = S::M, WT = S::WT, kRow = S::kRow;
    // Weights are 2^(logit - m).  The reference m lies kOff below the running
    // maximum when it is set, and is set again once the maximum is kOff + kSlack
    // above it (rescaling the sums of 16 rows at every new maximum of one of them
    // took a quarter of the instructions): weights are at most 2^15 in fp16, where
    // small ones stay normal and those below 2^-25, 2^-36 of the largest, are lost.  The product logit = x scale is rounded with the
    // difference, so a weight's exponent is off by up to half an ulp of m, which for
    // logits from kHuge on (an ulp of 1/2) counts in whole powers of two: those
    // are rounded first, and their m is the maximum itself.
    constexpr float kSlack = 4.0f, kOff = BF ? 0.0f : 11.0f, kHuge = 4194304.0f;
    __shared__ __attribute__((aligned(1024))) uint8_t mem[S::kLds];
    __shared__ float2 ml[WT][M];
    __shared__ typename std::conditional<kTurned, DecodeTables, Nothing>::type tab;
    __shared__ typename std::conditional<kTurned, TokenScales, Nothing>::type tscs[S::kBufs];

    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, gq = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wv % WR, wt = wv / WR;
    const PageGeom& g = a.g;
    const uint32_t mem0 = (uint32_t)(uintptr_t)(lds_u8*)mem;
    // Chunks of a token group's rows lie in 16-byte pieces exchanged by an
    // exclusive or with the row: the 16 rows that a load touches at one column
    // are in different banks.
    const auto swz = [](int row) { return D == 128 ? row & 15 : (row >> 1) & 7; };
    const uint32_t k_at = mem0 + (wt * T + i) * kRow + ((gq ^ swz(i)) * 16);
    const int vrow = 4 * gq + (i >> 2);
    const uint32_t v_at = mem0 + (wt * T + vrow) * kRow + ((((i >> 1) & 1) ^ swz(vrow)) * 16) + (i & 1) * 8;

    SeqBlock sb;
    int total, mine = 0;
    if (a.seqs <= 64) {
        sb = load_seqs(a, tl, 0, 0, lane, total);
    } else {
        sb = SeqBlock{-1, 0, 0, 0, 0, 0, 0, 0};
        total = block_sums(a, tl, lane, mine);
    }
    if constexpr (kTurned) {
        const int lo = tid & 15, hi = tid >> 4 & 15;  // (the second 256 threads write the same)
        tab.v[tid & 255] = pack2<false>(kAlphaV * pick(kV4, lo), kAlphaV * pick(kV4, hi));
        if constexpr (FMT == kMse) {
            const float x = pick(kV4, lo), y = pick(kV4, hi);
            const uint32_t h = pack2<false>(x, y);
            tab.k[tid & 255] = make_uint2(h, pack2<false>(x - h2f(h & 0xffff), y - h2f(h >> 16)));
        } else {
            const auto entry = [](int n) {
                return (__float_as_uint(pick(kK3, n & 7)) & ~1u) | (n & 8 ? 0u : 1u);
            };
            tab.k[tid & 255] = make_uint2(entry(lo), entry(hi));
        }
    }

    const Plan plan = make_plan(a, tl, total);
    const int all = plan.total * g.H;
    const long long begin = (long long)blockIdx.x * plan.per;
    const int stop = (int)min(begin + plan.per, (long long)all);

    // Bytes that can always be read, as an offset from the pool: the query's.
    const uint64_t dummy = (uint64_t)(reinterpret_cast<uintptr_t>(a.query) - reinterpret_cast<uintptr_t>(a.pool));

    bool first = true;
    for (int at = (int)min(begin, (long long)all); at < stop;) {
        const Piece pc = locate(a, tl, plan, at, lane, mine, sb);
        const int upto = min(pc.chunk + (stop - at), pc.chunks);
        const int c0 = max(pc.chunk - kLead, 0), c1 = upto - kLead;
        at += upto - pc.chunk;
        if (c1 <= c0) break;  // (the next workgroup has the item's tokens)
        const bool whole = c1 - c0 == pc.chunks - kLead;
        const int R = pc.rows * a.group, h = pc.h;
        const int32_t* __restrict__ table = a.tables + (size_t)pc.s * a.max_blocks;
        __syncthreads();  // the last piece's LDS is free (and the tables are written)

        // This lane's query rows: their tokens (the last row's past the item's end).
        int tok[RT];
        const auto row_of = [&](int rt) { return pc.tile * M + (wr * RT + rt) * 16 + i; };
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) tok[rt] = min(row_of(rt), R - 1) / a.group;
        const auto row_at = [&](int row, int token) {
            return ((size_t)(pc.row0 + token) * a.hq + h * a.group + (row - token * a.group)) * D;
        };
        const auto token_of = [&](int c) { return c * C + wt * T + (lane & (T - 1)); };
        const auto page_of = [&](int t, int& tib) {
            const int tc = max(min(t, pc.end - 1), 0);
            const int pg = g.bs_shift >= 0 ? tc >> g.bs_shift : tc / g.block_size;
            tib = tc - pg * g.block_size;
            return pg;
        };
        int tib;
        int id = table[page_of(token_of(c0), tib)], id2 = -1;
        constexpr bool kPair = WR > 1 && WT > 1;
        if (kPair) id2 = table[page_of(token_of(c0) + (wt ? -T : T), tib)];
        const auto readable = [&](int t, int pid) { return t < pc.end && pid >= 0; };

        // Compressed pages: the codes and scales of this lane's units of the
        // next chunk (unit u: a part of the codes of token u / kParts).
        constexpr int KU = kTurned ? S::KU : 1, kUnit = S::kUnit, kParts = S::kParts;
        typedef uint32_t code_t __attribute__((ext_vector_type(kUnit / 4), aligned(2)));
        code_t kc[KU], vc[KU];
        uint16_t ks[KU], kr[KU], vs[KU];
        int uid[KU];
        const auto unit_of = [&](int k) { return (wr + k * WR) * 64 + lane; };
        const auto unit_token = [&](int c, int k) { return c * C + wt * T + unit_of(k) / kParts; };
        const auto unit_ids = [&](int c) {
            if constexpr (kTurned) {
#pragma unroll
                for (int k = 0; k < KU; ++k) {
                    int tb;
                    uid[k] = table[page_of(unit_token(c, k), tb)];
                }
            }
        };
        const auto fetch = [&](int c) {
            if constexpr (kTurned) {
#pragma unroll
                for (int k = 0; k < KU; ++k) {
                    int tb;
                    const int t = unit_token(c, k);
                    (void)page_of(t, tb);
                    const bool ok = readable(t, uid[k]);
                    const uint64_t page = (uint64_t)max(uid[k], 0) * g.page_size;
                    const uint64_t cell = (uint64_t)(tb * g.H + h);
                    const int part = lane % kParts * kUnit;
                    const auto at_of = [&](uint64_t off, uint64_t n) {
                        return a.pool + (ok ? page + off + cell * n : dummy);
                    };
                    kc[k] = *reinterpret_cast<const code_t*>(at_of(g.kc_off, D / 2) + part);
                    vc[k] = *reinterpret_cast<const code_t*>(at_of(g.vc_off, D / 2) + part);
                    ks[k] = ld_u16(at_of(g.ks_off, 2));
                    if (FMT == kProd) kr[k] = ld_u16(at_of(g.kres_off, 2));
                    vs[k] = ld_u16(at_of(g.vs_off, 2));
                }
            }
        };
        const auto decode = [&](int buf) {
            if constexpr (kTurned) {
                auto& tsc = tscs[buf];
#pragma unroll
                for (int k = 0; k < KU; ++k) {
                    const int r = unit_of(k) / kParts;  // token of the group
                    const int part = lane % kParts;
                    if (part == 0) tsc.k[wt * T + r] = h2f(ks[k]);
                    if (part == 1) {
                        const float v = h2f(vs[k]);
                        tsc.v[wt * T + r] = v;
                        tsc.lv[wt * T + r] = fmaxf(log2_hw(fabsf(v)), -25.0f);
                    }
                    uint8_t* to = mem + buf * S::kTiles * S::kTile + (wt * T + r) * kRow;
                    const float re = FMT == kProd ? h2f(kr[k]) : 0.0f;
                    // A code dword (8 values) at a time; the next one's table entries are
                    // on their way meanwhile (each lookup waited for its own otherwise).
                    uint2 ke[2][4];
                    uint32_t ve[2][4];
                    const auto look_up = [&](int q) {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            ke[q & 1][b] = tab.k[kc[k][q] >> (8 * b) & 255];
                            ve[q & 1][b] = tab.v[vc[k][q] >> (8 * b) & 255];
                        }
                    };
                    look_up(0);
#pragma unroll
                    for (int q = 0; q < kUnit / 4; ++q) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (q + 1 < kUnit / 4) look_up(q + 1);
                        __builtin_amdgcn_sched_barrier(0);
                        u4 v, hi, lo;
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const uint2 e = ke[q & 1][b];
                            v[b] = ve[q & 1][b];
                            if constexpr (FMT == kMse) {
                                hi[b] = e.x;
                                lo[b] = e.y;
                            } else {  // level + (sign ? re : -re), 2^-24 of the level off
                                const uint2 w = split_k3(e, re);
                                hi[b] = w.x;
                                lo[b] = w.y;
                            }
                        }
                        const int piece = ((part * (kUnit / 4) + q) ^ swz(r)) * 16;
                        *reinterpret_cast<u4*>(to + piece) = hi;
                        *reinterpret_cast<u4*>(to + S::kTile + piece) = lo;
                        *reinterpret_cast<u4*>(to + 2 * S::kTile + piece) = v;
                    }
                }
            }
        };
        // Dense pages: the group's rows of chunk c straight into buffer c % 2.
        const auto stage = [&](int c, int pid) {
            if constexpr (!kTurned) {
                int tb;
                const int t = token_of(c);
                (void)page_of(t, tb);
                const uint64_t off = readable(t, pid)
                                         ? (uint64_t)pid * g.page_size + g.kc_off +
                                               (uint64_t)(tb * g.H + h) * kRow
                                         : dummy;
                const int off_lo = (int)(uint32_t)off, off_hi = (int)(off >> 32);
                constexpr int kRows = 1024 / kRow;  // rows of one load
                const uint32_t to = mem0 + (c & 1) * 2 * S::kTile + (wt * T + wr * (T / WR)) * kRow;
#pragma unroll
                for (int k = 0; k < T / WR / kRows; ++k) {
                    const int r = wr * (T / WR) + k * kRows + lane / (kRow / 16);
                    const uint64_t o = (uint64_t)(uint32_t)__shfl(off_lo, r, 64) |
                                       (uint64_t)(uint32_t)__shfl(off_hi, r, 64) << 32;
                    const int piece = ((lane % (kRow / 16)) ^ swz(r)) * 16;
                    const uint64_t ov = o == dummy ? dummy : o + (g.vc_off - g.kc_off);
                    load_to_lds(a.pool + o + piece, to + k * 1024);
                    load_to_lds(a.pool + ov + piece, to + S::kTile + k * 1024);
                }
            }
        };

        unit_ids(c0);
        // Query operands; the first chunk is on its way before they are prepared.
        constexpr int KK = D / 32;
        u4 qh[RT][KK], ql[kTurned ? RT : 1][KK];
        float qs[RT];
        u4 raws[RT][KK];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                raws[rt][kk] = *reinterpret_cast<const u4*>(a.query + row_at(min(row_of(rt), R - 1), tok[rt]) +
                                                            kk * 32 + gq * 8);
        stage(c0, id);
        fetch(c0);
        int next = id, next2 = id2;
        if (c0 + 1 < c1) {
            next = table[page_of(token_of(c0 + 1), tib)];
            if (kPair) next2 = table[page_of(token_of(c0 + 1) + (wt ? -T : T), tib)];
            unit_ids(c0 + 1);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const u4(&raw)[KK] = raws[rt];
            qs[rt] = scale;
            if constexpr (!kTurned) {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) qh[rt][kk] = raw[kk];
            } else {
                // q's rotation H (q s) as a product.  Row i of tile dt is dim 32 (dt / 2)
                // + 8 (i / 4) + 4 (dt % 2) + i % 4, so that a lane's results of tiles 2 kk
                // and 2 kk + 1 are the operand's dims 32 kk + 8 gq + 0..7; it holds
                // (-1)^(popcount(row & d) + d + h) at d = 32 kk + 8 gq + e: one pattern of e
                // for even and one for odd dt per lane, negated by kk and dt alone.
                uint32_t sg[2][4];
                const int par = h ^ __popc((i >> 2) & gq);
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const uint32_t s0 = (__popc((4 * k + (i & 3)) & e) ^ par) & 1;
                        const uint32_t s1 = (__popc((4 * k + (i & 3)) & (e + 1)) ^ par ^ 1) & 1;
                        sg[k][e / 2] = 0x3c003c00u | s0 << 15 | s1 << 31;
                    }
                f4 x[D / 16];
                float top = 0.0f;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    x[dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk) {
                        const uint32_t flip = __builtin_popcount((dt >> 1) & kk) & 1 ? 0x80008000u : 0u;
                        const uint32_t(&p)[4] = sg[dt & 1];
                        x[dt] = mfma<false>(u4{p[0] ^ flip, p[1] ^ flip, p[2] ^ flip, p[3] ^ flip}, raw[kk], x[dt]);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(x[dt][r]));
                }
                top = lane_xor_reduce<16>(top, [](float u, float w) { return fmaxf(u, w); });
                top = lane_xor_reduce<32>(top, [](float u, float w) { return fmaxf(u, w); });
                // A power of two brings the row's largest value into [2^13, 2^14),
                // so hi + lo keep 22 bits of it and no row leaves fp16's range.
                const int ex = (int)(__float_as_uint(top) >> 23) - 127;
                const int sh = top > 0.0f && ex < 128 ? 13 - max(ex, -100) : 0;
                const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
                qs[rt] = scale * inv * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float u = x[dt][2 * e] * up, w = x[dt][2 * e + 1] * up;
                        const uint32_t p = pack2<false>(u, w);
                        qh[rt][dt / 2][(dt & 1) * 2 + e] = p;
                        ql[rt][dt / 2][(dt & 1) * 2 + e] = pack2<false>(u - h2f(p & 0xffff), w - h2f(p >> 16));
                    }
            }
        }

        float m[RT], l[RT];
        f4 o[RT][D / 16];
        uint32_t plus[RT] = {}, minus[RT] = {};  // sums that hold +infinity, -infinity (bit dt * 4 + r)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        bool search = false;  // every chunk's values for infinities (see its end)
        for (int c = c0; c < c1; ++c) {
            const int tb0 = c * C + wt * T;  // the wave's first token
            constexpr uint64_t kAll = T == 64 ? ~0ull : (1ull << (T & 63)) - 1;
            const uint64_t live = __ballot(readable(token_of(c), id)) & kAll;
            const bool plain = !search && live == kAll && tb0 + T <= pc.L;
            // (the same in every wave: two token groups know each other's tokens)
            bool plain_all = plain;
            if constexpr (WR > 1 && WT > 1) {
                static_assert(WT == 2, "two token groups");
                const uint64_t other = __ballot(readable(token_of(c) + (wt ? -T : T), id2)) & kAll;
                plain_all = !search && live == kAll && other == kAll && c * C + C <= pc.L;
            }
            // The chunk's tiles are in LDS: loaded by its waves, or decoded now.  (A
            // wave's issue priority: products before softmax before decode, so that a
            // SIMD's waves take turns at matrix and vector instructions: 48.2 -> 45.7 us
            // for 32 sequences of up to 8,192 tokens, turbo_prod.  Two waves per SIMD
            // on dense pages gained nothing from it.)
            if constexpr (kTurned) {
                __builtin_amdgcn_s_setprio(0);
                decode(c & (S::kBufs - 1));
            } else {
                wait_vmem();
            }
            if constexpr (WR > 1) {
                __syncthreads();
            } else {
                // (the wave's own tiles: its last reads of the buffer that is
                // loaded next have arrived, its decoded values are written)
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            id = next;
            id2 = next2;
            if (c + 1 < c1) {
                stage(c + 1, next);
                fetch(c + 1);
                if (c + 2 < c1) {
                    next = table[page_of(token_of(c + 2), tib)];
                    if (kPair) next2 = table[page_of(token_of(c + 2) + (wt ? -T : T), tib)];
                    unit_ids(c + 2);
                }
            }
            const uint32_t kb = k_at + (c & (S::kBufs - 1)) * S::kTiles * S::kTile;
            const uint32_t vb = v_at + ((c & (S::kBufs - 1)) * S::kTiles + S::kTiles - 1) * S::kTile;
            const auto& tsc = tscs[c & (S::kBufs - 1)];

            const auto values = [&](int st, int dt) {
                const uint32_t p = (vb ^ (dt * 32)) + st * 32 * kRow;
                const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)p);
                const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(p + 16 * kRow));
                const u2 w0 = __builtin_bit_cast(u2, v0), w1 = __builtin_bit_cast(u2, v1);
                return u4{w0[0], w0[1], w1[0], w1[1]};
            };
            // The tokens that each row sees.
            uint64_t see[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) see[rt] = live;
            if (!plain) {
                const int j0 = tb0 - pc.L;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (j0 + T > 0) {  // (words before the drafted tokens: the prefix)
                        const int w0 = j0 >> 5;
                        const int32_t* mrow = a.mask + (size_t)(pc.row0 + tok[rt]) * a.mask_words;
                        uint32_t w[3];
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            w[k] = w0 + k < 0 ? ~0u : w0 + k < a.mask_words ? (uint32_t)mrow[w0 + k] : 0u;
                        const int sh = j0 & 31;
                        const uint32_t b0 = (uint32_t)(((uint64_t)w[1] << 32 | w[0]) >> sh);
                        const uint32_t b1 = (uint32_t)(((uint64_t)w[2] << 32 | w[1]) >> sh);
                        see[rt] &= (uint64_t)b1 << 32 | b0;
                    }
                }
            }
            // Dense pages hold any bits, also where a row sees nothing, and 0 * NaN is
            // NaN: a chunk with masked tokens is searched for infinities and NaN.
            // Where a row sees one (counted by a product of ones) its sums are
            // marked; then the values become zeros.
            if constexpr (!kTurned) {
                if (WR > 1 ? !plain_all : !plain) {
                    const uint32_t tile = mem0 + ((c & 1) * 2 + 1) * S::kTile +
                                          (WR > 1 ? wv * (S::kTile / NW) : wt * T * kRow) + lane * 16;
                    constexpr int kLoads = (WR > 1 ? S::kTile / NW : T * kRow) / 1024;
                    uint32_t bad = 0;
#pragma unroll 4
                    for (int k = 0; k < kLoads; ++k) {
                        const u4 w = *(lds_u4*)(uintptr_t)(tile + k * 1024);
#pragma unroll
                        for (int e = 0; e < 4; ++e) bad |= not_finite<BF>(w[e]);
                    }
                    const bool odd = WR > 1 ? __syncthreads_or(bad != 0) : __ballot(bad != 0) != 0;
                    if (odd) {
                        constexpr uint32_t one = BF ? 0x3f80u : 0x3c00u;
#pragma unroll 1
                        for (int dt = 0; dt < T / 32 * (D / 16); ++dt) {
                            const int st = dt / (D / 16), dd = dt % (D / 16);
                            const u4 v = values(st, dd);
                            u4 pos, neg;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                pos[e] = infinite_ones<BF>(v[e], 0u);
                                neg[e] = infinite_ones<BF>(v[e], 1u);
                            }
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                u4 ones;
                                const uint32_t sees = (uint32_t)(see[rt] >> (st * 32)) >> (gq * 4);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t b = sees >> ((e >> 1) * 16 + (e & 1) * 2);
                                    ones[e] = (b & 1 ? one : 0u) | (b & 2 ? one << 16 : 0u);
                                }
                                const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                                const f4 np = mfma<BF>(pos, ones, zero), nn = mfma<BF>(neg, ones, zero);
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    if (np[r] > 0.0f) plus[rt] |= 1u << (dd * 4 + r);
                                    if (nn[r] > 0.0f) minus[rt] |= 1u << (dd * 4 + r);
                                }
                            }
                        }
                        if (WR > 1) __syncthreads();
#pragma unroll 1
                        for (int k = 0; k < kLoads; ++k) {
                            u4 w = *(lds_u4*)(uintptr_t)(tile + k * 1024);
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] &= ~not_finite<BF>(w[e]);
                            *(lds_u4*)(uintptr_t)(tile + k * 1024) = w;
                        }
                        if (WR > 1) __syncthreads();
                    }
                }
            }

            // 32 tokens at a time: a row's logits, their weights, the values.
#pragma unroll 1
            for (int st = 0; st < T / 32; ++st) {
                const uint32_t ks_at = kb + st * 32 * kRow;
                const int tk = wt * T + st * 32 + gq * 4;  // this lane's tokens: tk + 16 ns + 0..3
                f4 x[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) x[rt][0] = x[rt][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                // K's operands are on their way before the products that take them, V's
                // before the softmax: left to the scheduler each product waited for its
                // own load.  (Independent sums next to each other: a product's result
                // is ready for the next of its own sum some products later.)
                u4 va[D / 16];
                if constexpr (kTurned) {
                    __builtin_amdgcn_s_setprio(2);
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns)
#pragma unroll
                        for (int kk = 0; kk < KK; ++kk) {
                            const u4 k0 = *(lds_u4*)(uintptr_t)((ks_at ^ (kk * 64)) + ns * 16 * kRow);
                            const u4 k1 = *(lds_u4*)(uintptr_t)((ks_at ^ (kk * 64)) + S::kTile + ns * 16 * kRow);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) x[rt][ns] = mfma<false>(k0, ql[rt][kk], x[rt][ns]);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) x[rt][ns] = mfma<false>(k1, qh[rt][kk], x[rt][ns]);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) x[rt][ns] = mfma<false>(k0, qh[rt][kk], x[rt][ns]);
                        }
                } else {
                    u4 k0[KK][2];
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                        for (int ns = 0; ns < 2; ++ns)
                            k0[kk][ns] = *(lds_u4*)(uintptr_t)((ks_at ^ (kk * 64)) + ns * 16 * kRow);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                        for (int ns = 0; ns < 2; ++ns)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) x[rt][ns] = mfma<BF>(k0[kk][ns], qh[rt][kk], x[rt][ns]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt) va[dt] = values(st, dt);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // Compressed pages: K's scale per token.  (The row's factor to a logit in
                // units of log2, above zero, enters below.)
                if constexpr (kTurned) {
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns) {
                        const f4 sk = *reinterpret_cast<const f4*>(&tsc.k[tk + ns * 16]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[rt][ns][r] *= sk[r];
                    }
                }
                if constexpr (kTurned) {
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_setprio(1);
                }
                uint32_t sees[RT];
                if (!plain) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        sees[rt] = (uint32_t)(see[rt] >> (st * 32)) >> (gq * 4);
#pragma unroll
                        for (int ns = 0; ns < 2; ++ns)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (!(sees[rt] >> (ns * 16 + r) & 1)) x[rt][ns][r] = -INFINITY;
                    }
                }
                // Running maximum.  Compressed pages: of logit + log2 |V's scale|, so
                // that the weights times their scales, what PV takes, are at most 2^15
                // whatever the scales are (-25: scales of zero take part too).
                float top[RT], ref[RT], to_log[RT];  // (x to_log: the logit)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) top[rt] = -INFINITY;
#pragma unroll
                for (int ns = 0; ns < 2; ++ns) {
                    f4 lv = {0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (kTurned) lv = *reinterpret_cast<const f4*>(&tsc.lv[tk + ns * 16]);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            top[rt] = fmaxf(top[rt], kTurned ? fmaf(x[rt][ns][r], qs[rt], lv[r]) : x[rt][ns][r]);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float t = kTurned ? top[rt] : top[rt] * scale;
                    t = lane_xor_reduce<16>(t, [](float u, float w) { return fmaxf(u, w); });
                    t = lane_xor_reduce<32>(t, [](float u, float w) { return fmaxf(u, w); });
                    to_log[rt] = kTurned ? qs[rt] : scale;
                    if (__ballot(t > m[rt] + (kOff + kSlack) || fabsf(t) >= kHuge)) {
                        const bool huge = fabsf(t) >= kHuge;
                        if (__ballot(huge)) {
                            // (V's scale is lost in the sum t; without it a weight is at
                            // most 1, its product with a scale at most 65,504)
                            float y = -INFINITY;
#pragma unroll
                            for (int ns = 0; ns < 2; ++ns)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    x[rt][ns][r] *= huge ? to_log[rt] : 1.0f;
                                    y = fmaxf(y, x[rt][ns][r]);
                                }
                            y = lane_xor_reduce<16>(y, [](float u, float w) { return fmaxf(u, w); });
                            y = lane_xor_reduce<32>(y, [](float u, float w) { return fmaxf(u, w); });
                            t = huge ? y : t;
                            to_log[rt] = huge ? 1.0f : to_log[rt];
                        }
                        const bool up = t > m[rt] + (huge ? 0.0f : kOff + kSlack);
                        const float mn = up ? t - (huge ? 0.0f : kOff) : m[rt];
                        const float f = up ? exp2_hw(m[rt] - mn) : 1.0f;
                        m[rt] = mn;
                        l[rt] *= f;
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] *= f;
                    }
                    ref[rt] = m[rt] == -INFINITY ? 0.0f : -m[rt];
                }
                u4 pw[RT], pl[RT];
                const auto weights = [&](auto masked) {
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns) {
                        f4 sv = {1.0f, 1.0f, 1.0f, 1.0f};
                        if constexpr (kTurned) sv = *reinterpret_cast<const f4*>(&tsc.v[tk + ns * 16]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            float p[4], sum = 0.0f;
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                p[r] = exp2_hw(fmaf(x[rt][ns][r], to_log[rt], ref[rt]));
                                sum += p[r];
                                if constexpr (kTurned) {
                                    p[r] *= sv[r];  // (not 0 * NaN where the row sees nothing)
                                    if (masked && !(sees[rt] >> (ns * 16 + r) & 1)) p[r] = 0.0f;
                                }
                            }
                            l[rt] += sum;
#pragma unroll
                            for (int r = 0; r < 4; r += 2) {
                                const uint32_t hi = pack2<BF>(p[r], p[r + 1]);
                                pw[rt][ns * 2 + r / 2] = hi;
                                pl[rt][ns * 2 + r / 2] = pack2_rest<BF>(hi, p[r], p[r + 1]);
                            }
                        }
                    }
                };
                if (!kTurned || plain)
                    weights(std::false_type{});
                else
                    weights(std::true_type{});
                if constexpr (kTurned) {  // (registers for V only now)
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt) va[dt] = values(st, dt);
                }
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma<BF>(va[dt], pl[rt], o[rt][dt]);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma<BF>(va[dt], pw[rt], o[rt][dt]);
            }
            if (kTurned && WR > 1 && S::kBufs == 1) __syncthreads();  // the tiles are decoded again
            // Infinite times a weight's low part, or times a weight that is zero, may
            // be NaN where the sum is infinite.  Sums that are not finite at the end
            // begin again, with every chunk searched.
            if constexpr (!kTurned) {
                if (c + 1 == c1 && !search) {
                    float sum = 0.0f;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt)
                            sum += (o[rt][dt][0] + o[rt][dt][1]) + (o[rt][dt][2] + o[rt][dt][3]);
                    const bool odd = !(fabsf(sum) < INFINITY);
                    if (WR > 1 ? __syncthreads_or(odd) : __ballot(odd) != 0) {
                        search = true;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            m[rt] = -INFINITY;
                            l[rt] = 0.0f;
#pragma unroll
                            for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                        }
                        id = table[page_of(token_of(c0), tib)];
                        if (kPair) id2 = table[page_of(token_of(c0) + (wt ? -T : T), tib)];
                        stage(c0, id);
                        next = id;
                        next2 = id2;
                        if (c0 + 1 < c1) {
                            next = table[page_of(token_of(c0 + 1), tib)];
                            if (kPair) next2 = table[page_of(token_of(c0 + 1) + (wt ? -T : T), tib)];
                        }
                        c = c0 - 1;
                    }
                }
            }
        }

        // A row's sum over its four lanes.
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (!kTurned) {
                if (__ballot((plus[rt] | minus[rt]) != 0)) {
#pragma unroll
                    for (int k = 0; k < D / 4; ++k) {
                        if (plus[rt] >> k & 1) o[rt][k / 4][k % 4] += INFINITY;
                        if (minus[rt] >> k & 1) o[rt][k / 4][k % 4] -= INFINITY;
                    }
                }
            }
            l[rt] = lane_xor_reduce<16>(l[rt], [](float u, float w) { return u + w; });
            l[rt] = lane_xor_reduce<32>(l[rt], [](float u, float w) { return u + w; });
            if (kTurned && whole) {
                // Rotated back (the merge does it for pieces): value dt * 16 + gq * 4 + r.
                const float sh = ((h & 1) ? -inv : inv) * (1.0f / kAlphaV);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    f4 y = o[rt][dt];
                    const f4 z = {y[0] + y[1], y[0] - y[1], y[2] + y[3], y[2] - y[3]};
                    y = f4{z[0] + z[2], z[1] + z[3], z[0] - z[2], z[1] - z[3]};
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        float u = y[r], w = y[r + 1];
                        butterfly2<16>(u, w);
                        butterfly2<32>(u, w);
                        y[r] = u;
                        y[r + 1] = w;
                    }
                    o[rt][dt] = y;
                }
#pragma unroll
                for (int k = 1; k < D / 16; k <<= 1)
#pragma unroll
                    for (int dt = 0; dt < D / 16; ++dt)
                        if (!(dt & k)) {
                            const f4 u = o[rt][dt], w = o[rt][dt + k];
                            o[rt][dt] = u + w;
                            o[rt][dt + k] = u - w;
                        }
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
                    o[rt][dt] *= f4{sh, -sh, sh, -sh};
            }
        }
        // (what follows is computed here, not kept over the chunks in registers
        // that then overflow to memory)
        int etid = tid;
        asm volatile("" : "+v"(etid));
        const int ei = etid & 15, eg = (etid >> 4) & 3;
        const int piece = 2 * blockIdx.x + (first ? 0 : 1);
        float* po = ws + (size_t)piece * M * D;
        constexpr int DW = D / 16 / WT;
        const auto merge_at = [&](int w, int rt, int dt) {
            return ((((w * WR + wr) * RT + rt) * (D / 16) + dt) * 64 + (etid & 63)) * 16;
        };
        float2* pm = reinterpret_cast<float2*>(ws + (size_t)2 * tl.groups * M * D) + (size_t)piece * M;
        if constexpr (WT > 1) {
            // The token groups' parts of a row on one reference; each group then adds up
            // and stores its share of the values, DW of the D / 16 tiles.  (Values lie as
            // the lanes hold them.  Added up row by row, each value with its groups' factors,
            // this took 8.5 us where it takes 8.1: 5 drafted tokens over 1,143, fp16.)
            if (eg == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) ml[wt][(wr * RT + rt) * 16 + ei] = make_float2(m[rt], l[rt]);
            }
            __syncthreads();  // every wave is done with the tiles
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mm = -INFINITY, lsum = 0.0f;
                float2 e[WT];
#pragma unroll
                for (int w = 0; w < WT; ++w) {
                    e[w] = ml[w][(wr * RT + rt) * 16 + ei];
                    mm = fmaxf(mm, e[w].x);
                }
                // (an empty part holds zeros, but for a NaN logit)
                const auto part = [&](float x) { return x == -INFINITY ? 1.0f : exp2_hw(x - mm); };
#pragma unroll
                for (int w = 0; w < WT; ++w) lsum += e[w].y * part(e[w].x);
                const float f = part(m[rt]);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt)
                    *reinterpret_cast<f4*>(mem + merge_at(wt, rt, dt)) = o[rt][dt] * f;
                m[rt] = mm;
                l[rt] = lsum;
            }
            __syncthreads();
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int dd = 0; dd < DW; ++dd) {
                    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < WT; ++w)
                        y += *reinterpret_cast<const f4*>(mem + merge_at(w, rt, wt * DW + dd));
                    o[rt][dd] = y;
                }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = (wr * RT + rt) * 16 + ei, row = pc.tile * M + r;
            if (row >= R) continue;
            const int d0 = wt * DW * 16 + eg * 4;
            if (whole) {
                const float f = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
                uint16_t* to = a.out + row_at(row, row / a.group) + d0;
#pragma unroll
                for (int dd = 0; dd < DW; ++dd) {
                    const f4 y = o[rt][dd] * f;
                    *reinterpret_cast<u2*>(to + dd * 16) = u2{pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3])};
                }
            } else {
#pragma unroll
                for (int dd = 0; dd < DW; ++dd) *reinterpret_cast<f4*>(po + r * D + d0 + dd * 16) = o[rt][dd];
                if (wt == 0 && eg == 0) pm[r] = make_float2(m[rt], l[rt]);
            }
        }
        first = false;
    }
}

// Merge of the items that were cut: WAVES waves per query row, D / 4 lanes per
// piece of it; compressed pages' sums are rotated back here.  A wave per row where
// there are rows for every SIMD (32 sequences of 6 drafted tokens, up to 16 pieces
// per row: 12.0 -> 7.4 us), else four (1,024 rows of 64 pieces, 34 MB: 13.8 -> 6.6 us),
// or sixteen where rows are few and four waves would take four or more rounds of
// loads (48 rows of 256 pieces 8.9 -> 7.5 us, 128 of 128 8.9 -> 7.8, 128 of 192 under
// turbo_prod 12.0 -> 9.1; 256 rows of 131 pieces 8.1 -> 8.4).
constexpr int merge_threads(int waves) { return waves > 4 ? 64 * waves : 256; }
template <bool BF, bool TURNED, int D, int WAVES>
__global__ __launch_bounds__(merge_threads(WAVES)) void tree_merge_kernel(const TreeArgs a, const Tiling tl,
                                                         const float* __restrict__ ws, float inv) {
    constexpr int kLanes = D / 4, kSides = 64 * WAVES / kLanes, kRows = merge_threads(WAVES) / (64 * WAVES), kDeep = 4;
    __shared__ float2 sml[kRows][kSides];
    __shared__ f4 so[kRows][kSides][kLanes];
    const int lane = threadIdx.x & 63, mine = threadIdx.x / (64 * WAVES);
    const int flat = __builtin_amdgcn_readfirstlane(blockIdx.x * kRows + mine);
    if (flat >= a.tokens * a.hq) return;
    const int tok = flat / a.hq, qh = flat - tok * a.hq, h = qh / a.group;
    int total = 0, row0 = -1, before = 0, chunks = 1;
    const auto look = [&](const SeqBlock& b) {
        const uint64_t hit = __ballot(b.row0 <= tok && tok < b.row0 + b.rows);
        if (!hit || row0 >= 0) return;
        const int k = __ffsll((unsigned long long)hit) - 1;
        row0 = __builtin_amdgcn_readlane(b.row0, k);
        before = __builtin_amdgcn_readlane(b.before, k);
        chunks = __builtin_amdgcn_readlane(b.chunks, k);
    };
    if (a.seqs <= 64) {
        look(load_seqs(a, tl, 0, 0, lane, total));
    } else {
        int mine;
        const int all = block_sums(a, tl, lane, mine);
        // the last block whose first row is this token's or before it (sequences
        // without rows begin where the next one does)
        int from = 0;
        for (int f = 0; f < a.seqs; f += 4096) {
            const int s = f + lane * 64;
            const uint64_t low = __ballot(s < a.seqs && a.row_start[min(s, a.seqs - 1)] <= tok);
            if (low) from = f + (63 - __clzll((unsigned long long)low)) * 64;
        }
        const int step = 64 * span_of(a.seqs), k = from / step;
        total = __builtin_amdgcn_readlane(sum_up(mine) - mine, k);
        for (int f = k * step; f <= from; f += 64) {
            const SeqBlock b = load_seqs(a, tl, f, total, lane, total);
            if (f == from) look(b);
        }
        total = all;
    }
    if (row0 < 0) return;  // behind the last sequence
    const Plan p = make_plan(a, tl, total);
    const int rr = (tok - row0) * a.group + (qh - h * a.group);
    const int tile = rr >> tl.m_log, r = rr & ((1 << tl.m_log) - 1);
    const int from = h * total + before + tile * chunks;
    const int w0 = (from + kLead) / p.per, w1 = (from + chunks - 1) / p.per;
    if (w0 == w1 || w1 >= tl.groups) return;  // whole: written by the split kernel
    const size_t M = (size_t)1 << tl.m_log;
    const float2* pm = reinterpret_cast<const float2*>(ws + (size_t)2 * tl.groups * M * D);
    const int side = threadIdx.x % (64 * WAVES) / kLanes, d = threadIdx.x % kLanes;
    float mm = -INFINITY, lsum = 0.0f;
    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](float om, float ol, f4 v) {
        const float mn = fmaxf(mm, om);
        const float fo = mm == -INFINITY ? 1.0f : exp2_hw(mm - mn);
        const float fn = om == -INFINITY ? 1.0f : exp2_hw(om - mn);
        y = y * fo + v * fn;
        lsum = lsum * fo + ol * fn;
        mm = mn;
    };
    for (int w = w0 + side; w <= w1; w += kSides * kDeep) {
        float2 e[kDeep];
        f4 v[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const int u = min(w + k * kSides, w1);
            const size_t q = ((size_t)2 * u + (u == w0 && from > u * p.per ? 1 : 0)) * M + r;
            e[k] = pm[q];
            v[k] = *reinterpret_cast<const f4*>(ws + q * D + d * 4);
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
            if (w + k * kSides <= w1) add(e[k].x, e[k].y, v[k]);
    }
    so[mine][side][d] = y;
    if (d == 0) sml[mine][side] = make_float2(mm, lsum);
    if constexpr (WAVES > 1)
        __syncthreads();  // (one row per workgroup: all of it is here)
    else
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (side * kLanes >= 64) return;
    const int sides = min(kSides, w1 - w0 + 1);
    for (int s = 0; s < sides; s += 8) {
        float2 e[8];
        f4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int u = min(s + k, sides - 1);
            e[k] = sml[mine][u];
            v[k] = so[mine][u][d];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s + k < sides && s + k != side) add(e[k].x, e[k].y, v[k]);
    }
    y *= lsum == 0.0f ? 0.0f : 1.0f / lsum;
    if constexpr (TURNED) {  // value d * 4 + r; every side of the wave holds the row
        const float sh = ((h & 1) ? -inv : inv) * (1.0f / kAlphaV);
        const f4 z = {y[0] + y[1], y[0] - y[1], y[2] + y[3], y[2] - y[3]};
        y = f4{z[0] + z[2], z[1] + z[3], z[0] - z[2], z[1] - z[3]};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            y[r] = butterfly<1>(y[r], lane);
            y[r] = butterfly<2>(y[r], lane);
            y[r] = butterfly<4>(y[r], lane);
            y[r] = butterfly<8>(y[r], lane);
            if (D == 128) y[r] = butterfly<16>(y[r], lane);
        }
        y *= f4{sh, -sh, sh, -sh};
    }
    if (side) return;
    *reinterpret_cast<u2*>(a.out + (size_t)flat * D + d * 4) =
        u2{pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3])};
}

template <int FMT, int D, int RT, int WR, int NW>
void launch_shape(const TreeArgs& a, hipStream_t stream) {
    using S = Shape<FMT, D, RT, WR, NW>;
    const auto log2i = [](int x) { return __builtin_ctz((unsigned)x); };
    Tiling t;
    t.m_log = log2i(S::M);
    t.c_log = log2i(S::C);
    // The line's length is known to the device only; here its bound.
    const long long chunks = std::max<long long>(1, ((long long)a.max_kv + S::C - 1) / S::C) + kLead;
    const long long items =
        (((long long)a.tokens * a.group) / S::M + std::min(a.seqs, a.tokens)) * a.g.H;
    if (items * chunks >= (1LL << 31) - (1 << 24))
        throw Error("tree_attention: too many (row tile, token chunk) pairs (2^31)");
    t.groups = (int)std::max<long long>(
        1, std::min<long long>((long long)num_cus() * S::kPerCu, items * chunks));
    constexpr size_t kPiece = (size_t)S::M * (D + 2) * sizeof(float);
    const bool cut = chunks > 1 + kLead;  // an item of one chunk is never cut
    const WorkspaceTurn turn(stream);
    // (room for every later call of this head_dim: 131,072 partial rows)
    float* ws = static_cast<float*>(Scratch{}.get(stream, cut ? 2 * (size_t)t.groups * kPiece : 0, "tree attention",
                                                  4 * (size_t)num_cus() * 128 * (D + 2) * sizeof(float)));
    hipLaunchKernelGGL((tree_split_kernel<FMT, D, RT, WR, NW>), dim3(t.groups), dim3(64 * NW), 0, stream, a, t,
                       ws, 1.44269504f * inv_sqrt_d(D), inv_sqrt_d(D));
    check_launch("tree_attention_kernel");
    if (!cut) return;
    const unsigned rows = (unsigned)(a.tokens * a.hq);
    const auto merge = [&](auto waves) {
        constexpr int W = decltype(waves)::value, per = merge_threads(W) / (64 * W);
        hipLaunchKernelGGL((tree_merge_kernel<S::BF, S::kTurned, D, W>), dim3((rows + per - 1) / per),
                           dim3(merge_threads(W)), 0, stream, a, t, ws, inv_sqrt_d(D));
    };
    // Waves per row: see tree_merge_kernel.  (Pieces of an item, of average length.)
    const long long pieces = std::min<long long>(chunks, t.groups / items);
    if (rows >= 8u * num_cus())
        merge(std::integral_constant<int, 1>{});
    else if (rows < (unsigned)num_cus() && pieces * (D / 4) >= 4 * 1024)
        merge(std::integral_constant<int, 16>{});
    else
        merge(std::integral_constant<int, 4>{});
    check_launch("tree_attention_merge_kernel");
}

// Query rows per tile: those of an average sequence (a tile of more rows decodes
// or loads a chunk once for all of them; fewer rows leave its products empty).
template <int FMT, int D>
void launch_format(const TreeArgs& a, hipStream_t stream) {
    constexpr bool kTurned = FMT == kProd || FMT == kMse;
    const long long rows = ((long long)a.tokens * a.group + a.seqs - 1) / a.seqs;
    // Tiles of 16 rows: each wave has tokens of its own, so no barrier, the shortest way
    // from a sequence's length to its sums.  Split + merge in us, these against the tiles
    // below (16 query heads on 2 kv heads, head_dim 128 unless said):
    //  - up to 16 rows, where the others are half empty, at head_dim 64: 32 sequences of up
    //    to 16,384 tokens fp16 38.4 / 40.5, turbo_prod 37.4 / 52.4, turbo_mse 34.3 / 48.8;
    //  - the same at head_dim 128 while a CU's share of tokens is small (tokens x tiles x kv
    //    heads per CU in brackets): 8 of up to 8,192 17.2 / 18.5, 20.2 / 21.6, 19.4 / 20.1
    //    (512), 8 of up to 16,384 22.3 / 23.9, 29.7 / 30.6, 27.9 / 28.0 (1,024); beyond, level
    //    (16: 39.4 / 39.4, 45.1 / 44.7, 42.1 / 40.4; 2,047), and a sequence of far more rows
    //    than the others has half the tiles;
    //  - more rows load or decode the tokens once per tile, which the shorter way outweighs
    //    while that share is small.  fp16: 8 drafted tokens over 2,048 12.1 / 15.0 (64), 32
    //    over 6,500 24.2 / 29.7 (816), 4 x 8 over 8,000 21.5 / 22.8 (1,001), 16 x 3-4 over
    //    8,192 33.7 / 24.8 (2,046).  head_dim 64: 4 x 8 over 8,000 17.8 / 19.0 fp16, 19.2 /
    //    21.6 turbo_prod, 18.4 / 21.4 turbo_mse (1,001);
    //  - compressed pages at head_dim 128, whose decode is the longest, sooner: turbo_prod
    //    32 over 2,048 19.8 / 23.1 (260), 16 over 8,192 26.6 / 27.8 (513), 32 over 6,500
    //    33.4 / 32.0 (816), 32 over 8,192 39.8 / 34.0 (1,028); turbo_mse 25.0 / 27.6 (513), 31.2 /
    //    31.7 (816).  Two tiles, which one of 32 rows holds without loss: 4 x 2-3 over 2,000
    //    13.7 / 13.1, 8 over 2,048 of 32 / 8 heads 17.4 / 16.7.
    const long long tiles = (rows + 15) / 16, work = tiles * a.seqs * a.max_kv * a.g.H;
    const long long most = !kTurned || D == 64 || tiles == 1 ? 1024 : tiles == 2 ? 0 : 640;
    if ((D == 64 && tiles == 1) || work <= most * num_cus()) return launch_shape<FMT, D, 1, 1, 4>(a, stream);
    if (rows <= 32) return launch_shape<FMT, D, 1, 2, 4>(a, stream);
    // (compressed pages: 16 rows a wave leave registers, but for five at head_dim 128
    // that spill, for a third workgroup of the CU: 48.6 -> 45.7 us for 32 sequences of
    // up to 8,192 tokens)
    if (rows <= 64) return launch_shape<FMT, D, kTurned ? 1 : 2, kTurned ? 4 : 2, 4>(a, stream);
    if (rows <= 128) return launch_shape<FMT, D, 2, 4, 4>(a, stream);
    return launch_shape<FMT, D, 2, 8, 8>(a, stream);
}

void launch_tree(int fmt, const TreeArgs& a, hipStream_t stream) {
    if (a.g.D == 128) {
        switch (fmt) {
            case kFp16: return launch_format<kFp16, 128>(a, stream);
            case kBf16: return launch_format<kBf16, 128>(a, stream);
            case kProd: return launch_format<kProd, 128>(a, stream);
            default: return launch_format<kMse, 128>(a, stream);
        }
    }
    switch (fmt) {
        case kFp16: return launch_format<kFp16, 64>(a, stream);
        case kBf16: return launch_format<kBf16, 64>(a, stream);
        case kProd: return launch_format<kProd, 64>(a, stream);
        default: return launch_format<kMse, 64>(a, stream);
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
        if ((long long)tokens * hq > (1LL << 26) - 4)  // (the merge's grid: 2^32 threads less 256)
            throw Error(w + "num_tokens * num_q_heads must be at most 2^26 - 4");
        const uint64_t cells = (uint64_t)g.block_size * g.H;
        const auto outside = [&](uint64_t off, uint64_t size) {
            return off > g.page_size || cells * size > g.page_size - off;
        };
        if (outside(g.kc_off, g.code_stride) || outside(g.vc_off, g.code_stride) ||
            (fmt > kBf16 && (outside(g.ks_off, 2) || outside(g.vs_off, 2) ||
                             (fmt == kProd && outside(g.kres_off, 2)))))
            throw Error(w + "layout does not match cfg (a region ends past the page)");
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
        a.group = hq / g.H;
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
