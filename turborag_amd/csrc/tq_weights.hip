// tq_weights.hip — softmax weights of query rows on the tokens of paged caches,
// summed over a kv head's rows: what an eviction by accumulated attention goes by.
//
//   out[s][h][t] = decay in[s][h][t] + sum over rows r of 2^(x_rt - M_r) / l_r,
//   x_rt = log2(e) <q_r, k_t> / sqrt(D), M_r = max over t, l_r = sum of 2^(x_rt - M_r).
//
// No value is read.  A weight needs its row's M and l, so the tokens are gone over
// twice: the first launch takes K's products with the rows and leaves each chunk's
// (max, sum) of every row; the last one forms the weights and adds them up over the
// rows, always in the same order and without atomics.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tq_device.h"

namespace tq {
namespace {

using namespace dev;

// What the pages hold.
constexpr int kFp16 = 0, kBf16 = 1, kProd = 2, kMse = 3;

struct WeightArgs {
    const uint16_t* query;
    const uint8_t* pool;
    const int32_t *tables, *row_start, *prefix;
    const float* in;  // null: nothing is added to
    float* out;
    int64_t stride;  // of in and out, from one head's scores to the next
    float decay;
    PageGeom g;  // dense pages: kc_off and code_stride of fp16/bf16 rows
    int max_blocks, hq, group, seqs, tokens, max_kv, causal;  // group: query heads per kv head
    uint32_t group_mul, group_shift;  // of the division by it
    // The workspace.  A row's index is that of its query: token * hq + query head.
    int chunk;              // tokens of a statistic
    int row_split;          // workgroups that share a chunk's rows
    float* logits;          // [rows][logit_stride]: x, or null
    int64_t logit_stride;
    float2* part;           // [chunks][rows]: (max, sum) of a chunk
    float2* stat;           // [rows]: (M, 1 / l)
    const uint16_t* turned;  // [rows][2 D]: q rotated, hi and lo (compressed pages)
    const float* turned_scale;  // [rows]
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// C += A B, A [16 x 32] by rows, B [32 x 16] by columns: lane l holds row
// (column) l % 16, k = 8 (l / 16) + 0..7; of C column l % 16, rows
// 4 (l / 16) + 0..3.
template <bool BF>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0,
                                                      0);
}

// n / group, n < 2^31: with 2^(shift - 1) < group <= 2^shift and mul = ceil(2^(32 + shift) /
// group) - 2^32, n (2^32 + mul) / 2^(32 + shift) is n / group and less than 1 / group more.
__device__ __forceinline__ int over_group(const WeightArgs& a, int n) {
    return (int)((__umulhi((uint32_t)n, a.group_mul) + (uint32_t)n) >> a.group_shift);
}

// A sequence's rows and tokens, as far as the call's bounds allow.
struct Seq {
    int row0, rows, L, end;  // first token row, token rows, prefix, tokens that some row may see
};
__device__ __forceinline__ Seq seq_of(const WeightArgs& a, int s) {
    Seq q;
    q.row0 = min(max(a.row_start[s], 0), a.tokens);
    q.rows = max(min(a.row_start[s + 1], a.tokens) - q.row0, 0);
    q.L = min(max(a.prefix[s], 0), a.max_kv);
    q.end = min(q.L + (a.causal ? q.rows : 0), a.max_kv);
    return q;
}

// ---------------------------------------------------------------------------
// Codes -> fp16 operands.  A code's fp16 value is looked up byte by byte: v_perm_b32
// takes four bytes by four selectors out of an 8-entry table in two registers (no LDS:
// four lookups an instruction).  The eight codes of a dword come out as dims 0 2 | 4 6 |
// 1 3 | 5 7, the order that the rotated queries are stored in.
// ---------------------------------------------------------------------------
struct Bytes8 {
    uint32_t a, b;  // entries 0..3, 4..7
};
struct Halves8 {
    Bytes8 lo, hi;  // low and high bytes of eight fp16 values
};
constexpr uint16_t half_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
constexpr float half_rest(float x) { return x - (float)(_Float16)x; }
template <class F>
constexpr Halves8 halves8(F f) {
    Halves8 r{};
    for (int k = 0; k < 8; ++k) {
        const uint32_t v = half_bits(f(k));
        (k < 4 ? r.lo.a : r.lo.b) |= (v & 255) << (8 * (k & 3));
        (k < 4 ? r.hi.a : r.hi.b) |= (v >> 8) << (8 * (k & 3));
    }
    return r;
}
constexpr float k3_at(int k) { return kK3[k]; }
constexpr float k3_rest(int k) { return half_rest(kK3[k]); }
constexpr float v4_at(int k) { return kV4[8 + k]; }  // the upper half: V4[15 - c] = -V4[c]
constexpr float v4_rest(int k) { return half_rest(kV4[8 + k]); }
constexpr bool v4_symmetric() {
    for (int k = 0; k < 8; ++k)
        if (kV4[7 - k] != -kV4[8 + k]) return false;
    return true;
}
static_assert(v4_symmetric(), "a code's value is +- that of its mirror");

__device__ __forceinline__ uint32_t look(const Bytes8& t, uint32_t sel) {
    return __builtin_amdgcn_perm(t.b, t.a, sel);
}
// Byte planes -> fp16 pairs of bytes 0 1 and 2 3.
__device__ __forceinline__ uint32_t pair01(uint32_t hi, uint32_t lo) {
    return __builtin_amdgcn_perm(hi, lo, 0x05010400u);
}
__device__ __forceinline__ uint32_t pair23(uint32_t hi, uint32_t lo) {
    return __builtin_amdgcn_perm(hi, lo, 0x07030602u);
}

// turbo_prod: K3 level in two fp16 parts, and the residual's sign as +-1.
struct KeyParts {
    u4 hi, lo, sign;
};
template <int FMT>
__device__ __forceinline__ KeyParts decode8(uint32_t w) {
    KeyParts r;
    if constexpr (FMT == kProd) {
        constexpr Halves8 H = halves8(k3_at), R = halves8(k3_rest);
        const uint32_t e = w & 0x07070707u, o = w >> 4 & 0x07070707u;
        const uint32_t eh = look(H.hi, e), el = look(H.lo, e), oh = look(H.hi, o), ol = look(H.lo, o);
        r.hi = u4{pair01(eh, el), pair23(eh, el), pair01(oh, ol), pair23(oh, ol)};
        const uint32_t fh = look(R.hi, e), fl = look(R.lo, e), ph = look(R.hi, o), pl = look(R.lo, o);
        r.lo = u4{pair01(fh, fl), pair23(fh, fl), pair01(ph, pl), pair23(ph, pl)};
        // (bit 3 set: added; 0xbc00 is -1)
        const uint32_t se = (w << 4 & 0x80808080u) ^ 0xbcbcbcbcu, so = (w & 0x80808080u) ^ 0xbcbcbcbcu;
        const auto wide01 = [](uint32_t p) { return __builtin_amdgcn_perm(p, p, 0x010c000cu); };
        const auto wide23 = [](uint32_t p) { return __builtin_amdgcn_perm(p, p, 0x030c020cu); };
        r.sign = u4{wide01(se), wide23(se), wide01(so), wide23(so)};
    } else {
        constexpr Halves8 H = halves8(v4_at), R = halves8(v4_rest);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t n = (k ? w >> 4 : w) & 0x0f0f0f0fu;
            const uint32_t below = ~n & 0x08080808u, minus = below << 4;
            const uint32_t m = (n ^ (below - (below >> 3))) & 0x07070707u;  // of the upper half
            const uint32_t hh = look(H.hi, m) | minus, hl = look(H.lo, m);
            const uint32_t rh = look(R.hi, m) ^ minus, rl = look(R.lo, m);
            r.hi[2 * k] = pair01(hh, hl);
            r.hi[2 * k + 1] = pair23(hh, hl);
            r.lo[2 * k] = pair01(rh, rl);
            r.lo[2 * k + 1] = pair23(rh, rl);
        }
    }
    return r;
}

// ---------------------------------------------------------------------------
// Queries of compressed pages: q's rotation H (q s) in two fp16 parts, brought by a
// power of two to a largest value in [2^13, 2^14) (22 bits of it are kept and no row
// leaves fp16's range); D / 8 lanes a row, eight dims each.
// ---------------------------------------------------------------------------
struct Turned {
    u4 hi, lo;
    float unscale;  // undoes the power of two
};
template <int D>
__device__ __forceinline__ Turned turn_query(u4 raw, int h, int j) {
    constexpr int L = D / 8;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = h2f(raw[e / 2] >> (16 * (e & 1)) & 0xffff) * sign_of(e, h);
#pragma unroll
    for (int m = 1; m < 8; m <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!(e & m)) {
                const float u = x[e], v = x[e | m];
                x[e] = u + v;
                x[e | m] = u - v;
            }
#pragma unroll
    for (int m = 1; m < L; m <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float o = xor_lane(x[e], m);
            x[e] = j & m ? o - x[e] : x[e] + o;
        }
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
    top = max_lanes<L>(top);
    const int ex = (int)(__float_as_uint(top) >> 23) - 127;
    const int sh = top > 0.0f && ex < 128 ? 13 - max(ex, -100) : 0;
    const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
    Turned t;
#pragma unroll
    for (int p = 0; p < 4; ++p) {  // dims 0 2 | 4 6 | 1 3 | 5 7
        const int d = (p & 1) * 4 + (p >> 1);
        const float u = x[d] * up, v = x[d + 2] * up;
        t.hi[p] = f2h2(u, v);
        t.lo[p] = f2h2(u - h2f(t.hi[p] & 0xffff), v - h2f(t.hi[p] >> 16));
    }
    t.unscale = __uint_as_float((uint32_t)(127 - sh) << 23);
    return t;
}
// All rows, for the passes that go over more than a few.
template <int D>
__global__ __launch_bounds__(256) void turn_queries_kernel(const uint16_t* __restrict__ query, int hq, int group,
                                                           int rows, uint16_t* __restrict__ turned,
                                                           float* __restrict__ turned_scale, float scale) {
    constexpr int L = D / 8;
    const int j = threadIdx.x % L, at = blockIdx.x * (256 / L) + threadIdx.x / L;
    const int row = min(at, rows - 1);
    const u4 raw = *reinterpret_cast<const u4*>(query + (size_t)row * D + 8 * j);
    const Turned t = turn_query<D>(raw, row % hq / group, j);
    if (at != row) return;
    *reinterpret_cast<u4*>(turned + (size_t)row * 2 * D + 8 * j) = t.hi;
    *reinterpret_cast<u4*>(turned + (size_t)row * 2 * D + D + 8 * j) = t.lo;
    if (j == 0) turned_scale[row] = scale * t.unscale;
}

// (max, sum) of a part added to a row's.
__device__ __forceinline__ void add_part(float& m, float& l, float2 e) {
    const float n = fmaxf(m, e.x);
    l = (m == -INFINITY ? l : l * exp2_hw(m - n)) + (e.x == -INFINITY ? e.y : e.y * exp2_hw(e.x - n));
    m = n;
}

// ---------------------------------------------------------------------------
// K of a wave's 16 TT tokens of a sequence: lane (i, gq) has token i of each tile.
// ---------------------------------------------------------------------------
template <int FMT, int D, int TT>
struct Keys {
    static constexpr bool kTurned = FMT == kProd || FMT == kMse, BF = FMT == kBf16;
    static constexpr int KK = D / 32, T = 16 * TT;
    typedef uint32_t code_t __attribute__((ext_vector_type(KK), aligned(2)));
    int id[TT], tib[TT];
    uint32_t live[TT];                  // tokens of the tile that can be read (bits)
    u4 k[kTurned ? 1 : TT][KK];         // dense: operands
    code_t code[kTurned ? TT : 1];      // compressed: a quarter of a token's codes
    uint32_t scales[kTurned ? TT : 1];  // its RMS, its residual's RMS above
    float ks[kTurned ? TT : 1][4], kr[kTurned ? TT : 1][4];  // of the tokens 4 gq + 0..3

    __device__ __forceinline__ void pages(const WeightArgs& a, const int32_t* table, int t0, int end, int i) {
        const PageGeom& g = a.g;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = min(t0 + tt * 16 + i, end - 1);
            const int pg = g.bs_shift >= 0 ? t >> g.bs_shift : t / g.block_size;
            tib[tt] = t - pg * g.block_size;
            id[tt] = table[pg];
        }
    }
    // (what cannot be read comes from the query instead)
    __device__ __forceinline__ void fetch(const WeightArgs& a, int h, int t0, int end, int i, int gq) {
        const PageGeom& g = a.g;
        const uint64_t dummy = (uint64_t)(reinterpret_cast<uintptr_t>(a.query) - reinterpret_cast<uintptr_t>(a.pool));
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const bool ok = t0 + tt * 16 + i < end && id[tt] >= 0;
            live[tt] = (uint32_t)__ballot(ok) & 0xffffu;
            const uint64_t page = (uint64_t)max(id[tt], 0) * g.page_size;
            const uint64_t cell = (uint64_t)(tib[tt] * g.H + h);
            if constexpr (!kTurned) {
                const uint8_t* p = a.pool + (ok ? page + g.kc_off + cell * (2 * D) : dummy) + gq * 16;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) k[tt][kk] = *reinterpret_cast<const u4*>(p + kk * 64);
            } else {
                code[tt] = *reinterpret_cast<const code_t*>(
                    a.pool + (ok ? page + g.kc_off + cell * (D / 2) : dummy) + gq * (D / 8));
                scales[tt] = ld_u16(a.pool + (ok ? page + g.ks_off + cell * 2 : dummy));
                if (FMT == kProd)
                    scales[tt] |= (uint32_t)ld_u16(a.pool + (ok ? page + g.kres_off + cell * 2 : dummy)) << 16;
            }
        }
    }
    __device__ __forceinline__ void scales_of(int gq) {
        if constexpr (kTurned) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t w = (uint32_t)__shfl((int)scales[tt], 4 * gq + r, 64);
                    ks[tt][r] = h2f(w & 0xffff);
                    kr[tt][r] = FMT == kProd ? h2f(w >> 16) : 0.0f;
                }
            }
        }
    }
    // Every row sees all of them whose first L tokens it sees.
    __device__ __forceinline__ bool plain(int t0, int L) const {
        uint32_t all = 0xffffu;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) all &= live[tt];
        return all == 0xffffu && t0 + T <= L;
    }
    // Their products with N times 16 query rows: operand(n, part, piece) is a row's 16-byte
    // piece.  Compressed keys are decoded 32 dims at a time, for all the rows.
    template <int N, class Operand>
    __device__ __forceinline__ void products(f4 (&x)[N][TT], int gq, Operand&& operand) const {
        f4 y[N][TT];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) x[n][tt] = y[n][tt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (!kTurned) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                u4 q[KK];
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) q[kk] = operand(n, 0, kk * 4 + gq);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) x[n][tt] = mfma<BF>(k[tt][kk], q[kk], x[n][tt]);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                __builtin_amdgcn_sched_barrier(0);  // (no operands ahead: registers)
                KeyParts kp[TT];
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) kp[tt] = decode8<FMT>(code[tt][kk]);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const u4 qh = operand(n, 0, gq * KK + kk), ql = operand(n, 1, gq * KK + kk);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) x[n][tt] = mfma<false>(kp[tt].hi, qh, x[n][tt]);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
                        if (FMT == kProd) y[n][tt] = mfma<false>(kp[tt].sign, qh, y[n][tt]);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) x[n][tt] = mfma<false>(kp[tt].hi, ql, x[n][tt]);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
                        if (FMT == kProd) y[n][tt] = mfma<false>(kp[tt].sign, ql, y[n][tt]);
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) x[n][tt] = mfma<false>(kp[tt].lo, qh, x[n][tt]);
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (FMT == kProd) x[n][tt][r] = fmaf(kr[tt][r], y[n][tt][r], x[n][tt][r]);
                        x[n][tt][r] *= ks[tt][r];
                    }
        }
    }
    // -infinity for the tokens that a row of so many does not see.
    __device__ __forceinline__ void mask(f4 (&x)[TT], int t0, int limit, int gq) const {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = tt * 16 + 4 * gq + r;
                if (t0 + t >= limit || !(live[tt] >> (4 * gq + r) & 1)) x[tt][r] = -INFINITY;
            }
    }
};

// Tokens that a row sees.
__device__ __forceinline__ int limit_of(const WeightArgs& a, const Seq& q, int row) {
    return min(q.L + (a.causal ? over_group(a, row) + 1 : 0), a.max_kv);
}
__device__ __forceinline__ size_t query_row(const WeightArgs& a, const Seq& q, int h, int row) {
    const int tok = over_group(a, row);
    return (size_t)(q.row0 + tok) * a.hq + h * a.group + (row - tok * a.group);
}
// Rows lie in LDS in 16-byte pieces exchanged by an exclusive or with the row: the 16 rows
// that a load touches at one column are in different banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
    return D == 128 ? row & 15 : (row >> 1) & 7;
}
__device__ __forceinline__ float max_of(float u, float w) { return fmaxf(u, w); }
__device__ __forceinline__ float sum_of(float u, float w) { return u + w; }
// Over the four lanes that hold a row's tokens.
__device__ __forceinline__ float row_max(float m) {
    return lane_xor_reduce<32>(lane_xor_reduce<16>(m, max_of), max_of);
}
__device__ __forceinline__ float row_sum(float l) {
    return lane_xor_reduce<32>(lane_xor_reduce<16>(l, sum_of), sum_of);
}
template <int TT>
__device__ __forceinline__ float largest(const f4 (&x)[TT]) {
    float m = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
#pragma unroll
    for (int tt = 1; tt < TT; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, x[tt][r]);
    return m;
}

// ---------------------------------------------------------------------------
// The passes over K.  A workgroup has one kv head and a chunk of C tokens of one
// sequence; 4 groups of its waves have T tokens each at a time, whose K operands stay
// in registers while the rows go by in tiles of 16, dealt to WR waves; the rows'
// operands come from LDS, a block of kRowBlock rows at a time.  The products run
// transposed (K Q'): a query row is a lane column, so its maximum and sum are in-lane
// but for two lane swaps, and a token's sum over the rows is in-lane over the tiles,
// across 16 lanes once at the end.
//   kStats: (max, sum) of the chunk for every row;  kStore: x too;
//   kSum: the weights, summed over the rows.
// Blocks of few rows (of 16 at head_dim 128): compressed pages' queries are rotated here.
// kSplits: a.row_split workgroups share a chunk's blocks.
// Bound by: memory with few rows of dense pages (32 sequences, 540K tokens, 8 rows: 277 MB of
// K and 35 MB of x in 62.5 us, 5.0 TB/s); latency where a workgroup has one chunk and
// its rows (256 rows of 32K tokens: 17 us a launch, of which the products and exponentials
// are 5 to 6); for compressed pages latency at few waves, one chain page ids -> codes -> decode
// -> products after the other (64 rows of 32 sequences to 8K tokens: 39 us at two waves a SIMD,
// which issue in 41% of their cycles, wait for loads in 32% and for a free unit in 27%; vector
// units 34% busy, matrix cores 20%: five products where dense keys have one).  A key is decoded
// 32 dims at a time for all rows of a block, so that three or four waves of a SIMD have
// registers where rows are fewer (32 rows, 32 x 8K tokens: 51.6 -> 46.0 us with the sum).
// Rows that see nothing of a chunk are worked through as the others are: half of both passes
// for a whole prompt (2,048 tokens without a prefix 234 us, 8,192 3,039).
// ---------------------------------------------------------------------------
constexpr int kStats = 0, kStore = 1, kSum = 2;
template <int FMT, int D>
struct Blocks {  // rows of a block
    static constexpr int kFew = 2048 / D, kSmall = 4096 / D;
    static constexpr int kLarge = (FMT == kProd || FMT == kMse ? 8192 : 16384) / D;
};
// x rs, the logit in powers of two, is one number in both passes, whatever rows share a tile and
// whatever the row's maximum is there: exact below kHuge and rounded from there on (its difference
// from a rounded maximum may be above 0 by half an ulp of that, which would overflow).  A maximum
// of at least half of kHuge says that a tile may have such logits that count: those of a smaller
// maximum are at least 2^21 below it, 0 either way.  (An infinite one is a row that sees nothing,
// or one of NaN.)
constexpr float kHuge = 4194304.0f;
__device__ __forceinline__ bool near_huge(float m) { return fabsf(m) >= kHuge / 2 && fabsf(m) < INFINITY; }
__device__ __forceinline__ float over_huge(float x, float rs, float ref) {
    const float y = x * rs;
    return fabsf(y) >= kHuge ? y - ref : fmaf(x, rs, -ref);
}

template <int FMT, int D, int WT, int WR, int MODE, int RB>
struct Shape {
    static constexpr bool kTurned = FMT == kProd || FMT == kMse;
    // (compressed pages: three operands a token tile)
    static constexpr int TT = kTurned ? 2 : 4, T = 16 * TT, kSubs = kTurned ? 2 : 1, C = T * WT * kSubs;
    static constexpr int kParts = kTurned ? 2 : 1;  // of a query row
    static constexpr int kRowBytes = 2 * D;
    static constexpr bool kTurns = kTurned && MODE == kStore && RB == Blocks<FMT, D>::kFew;
    static constexpr int kRowBlock = RB, kPart = RB * kRowBytes;  // bytes of a block's part
    static constexpr bool kSplits = MODE != kSum && RB == Blocks<FMT, D>::kSmall;
    static constexpr int kThreads = 64 * WT * WR;
    static constexpr int kTiles = !kTurned ? 1 : RB >= 64 ? 4 : RB / 16;  // of rows that share a decoded key
    static constexpr int kWaves = kTurned ? (kTiles < 4 ? 5 - kTiles : 2) : MODE == kSum ? 2 : 3;  // of a SIMD, at least
};

template <int FMT, int D, int WT, int WR, int MODE, int RB>
__global__ __launch_bounds__(64 * WT * WR, (Shape<FMT, D, WT, WR, MODE, RB>::kWaves)) void weights_kernel(const WeightArgs a, float scale) {
    using S = Shape<FMT, D, WT, WR, MODE, RB>;
    constexpr bool kTurned = S::kTurned;
    constexpr int TT = S::TT, T = S::T, C = S::C, kRowBlock = S::kRowBlock;
    __shared__ __attribute__((aligned(16))) uint8_t rows_mem[S::kPart * S::kParts];
    __shared__ float row_scales[kTurned ? kRowBlock : 1];
    __shared__ float2 ml[MODE == kSum ? 1 : WT][kRowBlock];  // kSum: the rows' (M, 1 / l)
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, gq = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wv % WT, wr = wv / WT;
    const PageGeom& g = a.g;

    // Eight chunks in turn, then the same ones of the next head: the workgroups of one
    // chunk run on one XCD, whose L2 then holds the lines that the heads share.
    const int chunks = (a.max_kv + C - 1) / C;
    unsigned b = blockIdx.y * gridDim.x + blockIdx.x, part_of = 0;
    if (S::kSplits && a.row_split > 1) {
        const unsigned whole = ((unsigned)a.seqs * (unsigned)chunks + 7) / 8 * 8 * (unsigned)g.H;
        part_of = b / whole;
        b -= part_of * whole;
    }
    const unsigned eight = b / 8;
    const int h = (int)(eight % (unsigned)g.H);
    const long long sc = (long long)(eight / (unsigned)g.H) * 8 + b % 8;
    if (sc >= (long long)a.seqs * chunks || (S::kSplits && part_of >= (unsigned)a.row_split)) return;
    const int s = (int)(sc / chunks), c = (int)(sc - (long long)s * chunks);
    const Seq q = seq_of(a, s);
    if (c * C >= q.end) return;
    const int R = q.rows * a.group;
    if (R == 0) {  // (no row and, without any in the call, no query)
        const int64_t at = ((int64_t)s * g.H + h) * a.stride;
        if (MODE == kSum)
            for (int t = c * C + tid; t < min(c * C + C, q.end); t += S::kThreads)
                a.out[at + t] = a.in ? a.decay * a.in[at + t] : 0.0f;
        return;
    }

    const int32_t* __restrict__ table = a.tables + (size_t)s * a.max_blocks;
    Keys<FMT, D, TT> keys;
    const int first = c * C + wt * T;

    // The block's rows into LDS: on their way (in registers) while the block before is
    // worked on, the first one while K is.
    const auto nat_of = [&](int row) { return query_row(a, q, h, row); };
    const auto swz = [](int row) { return swizzle<D>(row); };
    constexpr int kPieces = S::kRowBytes / 16 * S::kParts, kHold = S::kTurns ? 1 : S::kPart * S::kParts / 16 / S::kThreads;
    u4 hold[kHold];
    float2 hold_stat;
    float hold_scale;
    const auto take = [&](int rb) {
        if constexpr (S::kTurns) {  // D / 8 lanes a row
            static_assert(kRowBlock * (D / 8) == S::kThreads, "a thread per eight dims of a block");
            hold[0] = *reinterpret_cast<const u4*>(a.query + nat_of(min(rb + tid / (D / 8), R - 1)) * D + tid % (D / 8) * 8);
            return;
        }
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
            const int x = k * S::kThreads + tid, p = x % kPieces;
            const size_t nat = nat_of(min(rb + x / kPieces, R - 1));
            hold[k] = *reinterpret_cast<const u4*>((kTurned ? a.turned : a.query) + nat * (S::kParts * D) + p * 8);
        }
        static_assert(kRowBlock <= S::kThreads, "a thread per row of a block");
        if (kTurned || MODE == kSum) {
            const size_t nat = nat_of(min(rb + tid, R - 1));
            if (kTurned) hold_scale = a.turned_scale[nat];
            if (MODE == kSum) hold_stat = a.stat[nat];
        }
    };
    const auto put = [&](int rb) {
        if constexpr (S::kTurns) {
            const int r = tid / (D / 8), p = tid % (D / 8);
            const Turned t = turn_query<D>(hold[0], h, p);
            uint8_t* to = rows_mem + r * S::kRowBytes + (p ^ swz(r)) * 16;
            *reinterpret_cast<u4*>(to) = t.hi;
            *reinterpret_cast<u4*>(to + S::kPart) = t.lo;
            if (p == 0) row_scales[r] = scale * t.unscale;
            return;
        }
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
            const int x = k * S::kThreads + tid, r = x / kPieces, y = x % kPieces;
            const int p = y % (S::kRowBytes / 16), part = y / (S::kRowBytes / 16);
            *reinterpret_cast<u4*>(rows_mem + part * S::kPart + r * S::kRowBytes + (p ^ swz(r)) * 16) = hold[k];
        }
        if (tid < kRowBlock) {
            if (kTurned) row_scales[tid] = hold_scale;
            if (MODE == kSum) ml[0][tid] = rb + tid < R ? hold_stat : make_float2(INFINITY, 0.0f);
        }
    };
    // (page ids first: K hangs on them)
    keys.pages(a, table, first, q.end, i);
    __builtin_amdgcn_sched_barrier(0);
    const int rb0 = S::kSplits ? (int)part_of * kRowBlock : 0, step = S::kSplits ? a.row_split * kRowBlock : kRowBlock;
    if (S::kSplits && rb0 >= R) return;
    take(rb0);

    float acc[S::kSubs][TT][4];
#pragma unroll
    for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[u][tt][r] = 0.0f;

    if (S::kSubs == 1) keys.fetch(a, h, first, q.end, i, gq);
    for (int rb = rb0; rb < R; rb += step) {
        const int n = min((R - rb + 15) & ~15, kRowBlock);
        if (rb != rb0) __syncthreads();
        if (kTurned && rb != rb0) take(rb);
        put(rb);
        __syncthreads();
        if (!kTurned && rb + step < R) take(rb + step);  // (those have no registers left)
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u) {
            const int t0 = first + u * WT * T;
            if (S::kSubs > 1) {
                if (rb != rb0 || u) keys.pages(a, table, t0, q.end, i);
                keys.fetch(a, h, t0, q.end, i, gq);
            }
            keys.scales_of(gq);
            const bool plain = keys.plain(t0, q.L);
            if (t0 >= q.end && (MODE == kSum || (MODE == kStats && u))) continue;

            constexpr bool kOnce = kTurned && 16 * S::kTiles == kRowBlock;
            static_assert(S::kTiles == 1 || WR == 1, "the tiles of a wave lie in a row");
            for (int r0 = wr * 16; r0 < n; r0 += 16 * WR * S::kTiles) {
                f4 xs[S::kTiles][TT];
                keys.products(xs, gq, [&](int k, int part, int piece) {
                    const int r = r0 + k * 16 + i;
                    return *reinterpret_cast<const u4*>(rows_mem + part * S::kPart + r * S::kRowBytes + (piece ^ swz(r)) * 16);
                });
#pragma unroll
                for (int k = 0; k < S::kTiles; ++k) {
                    if (k && r0 + 16 * k >= n) break;
                    f4(&x)[TT] = xs[k];
                    const int at = r0 + 16 * k + i, row = min(rb + at, R - 1);
                    // x rs: the logit in powers of two.
                    float rs = kTurned ? row_scales[at] : scale;
                    if (!plain) keys.mask(x, t0, limit_of(a, q, row), gq);
                    const auto differences = [&](float& ref) {  // into x, for fmaf(x, rs, -ref)
#pragma unroll
                        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[tt][r] = over_huge(x[tt][r], rs, ref);
                        rs = 1.0f;
                        ref = 0.0f;
                    };
                    if constexpr (MODE == kSum) {
                        float2 st = ml[0][at];
                        if (__ballot(near_huge(st.x))) differences(st.x);
#pragma unroll
                        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                acc[u][tt][r] = fmaf(exp2_hw(fmaf(x[tt][r], rs, -st.x)), st.y, acc[u][tt][r]);
                    } else {
                        if (MODE == kStore) {  // (rounded where it is stored)
#pragma unroll
                            for (int tt = 0; tt < TT; ++tt) x[tt] *= rs;
                            rs = 1.0f;
                        }
                        float m = row_max(largest(x)) * rs;
                        float ref = m == -INFINITY ? 0.0f : m;
                        if (MODE == kStats && __ballot(near_huge(m))) differences(ref);
                        float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) l4[r] += exp2_hw(fmaf(x[tt][r], rs, -ref));
                        float l = row_sum((l4[0] + l4[1]) + (l4[2] + l4[3]));
                        if (gq == 0) {
                            if (u) {  // (the wave's own entry)
                                const float2 e = ml[wt][at];
                                add_part(m, l, e);
                            }
                            ml[wt][at] = make_float2(m, l);
                        }
                        if constexpr (MODE == kStore) {
                            if (rb + at < R) {
                                float* to = a.logits + (int64_t)nat_of(row) * a.logit_stride + t0 + 4 * gq;
#pragma unroll
                                for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<f4*>(to + tt * 16) = x[tt];
                            }
                        }
                    }
                }
                if (kOnce) break;
            }
        }
        if constexpr (MODE != kSum) {
            __syncthreads();
            for (int r = tid; r < min(n, R - rb); r += S::kThreads) {
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < WT; ++w) m = fmaxf(m, ml[w][r].x);
#pragma unroll
                for (int w = 0; w < WT; ++w) {
                    const float2 e = ml[w][r];
                    l += e.x == -INFINITY ? e.y : e.y * exp2_hw(e.x - m);
                }
                a.part[(size_t)c * ((size_t)a.tokens * a.hq) + nat_of(rb + r)] = make_float2(m, l);
            }
        }
    }
    if constexpr (MODE == kSum) {
        // Over the lanes' rows, then over the waves that shared them.
        __syncthreads();
        float* sums = reinterpret_cast<float*>(rows_mem);  // [WR][C]
        const int64_t at = ((int64_t)s * g.H + h) * a.stride;
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                float mine = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = sum_lanes<16>(acc[u][tt][r]);
                    mine = i == r ? w : mine;
                }
                if (i < 4) sums[wr * C + u * WT * T + wt * T + tt * 16 + 4 * gq + i] = mine;
            }
        __syncthreads();
        static_assert(C <= S::kThreads, "a thread per token");
        const int t = c * C + tid;
        if (tid < C && t < q.end) {
            float w = sums[tid];
#pragma unroll
            for (int k2 = 1; k2 < WR; ++k2) w += sums[k2 * C + tid];
            a.out[at + t] = a.in ? fmaf(a.decay, a.in[at + t], w) : w;
        }
    }
}

// A row's (M, 1 / l); one that sees nothing gives every token 2^-infinity * 0.
__device__ __forceinline__ float2 row_stat(float m, float l) {
    return l == 0.0f ? make_float2(INFINITY, 0.0f) : make_float2(m, 1.0f / l);
}

// The last sequence that begins at or before token row `tok` (those without rows begin
// where the next one does); a wave together.
__device__ __forceinline__ int find_seq(const WeightArgs& a, int tok, int lane) {
    int lo = 0, span = a.seqs;
    while (span > 1) {
        const int step = (span + 63) / 64, at = lane * step;
        const uint64_t low = __ballot(at < span && a.row_start[lo + min(at, span - 1)] <= tok);
        const int k = max(63 - __clzll((unsigned long long)(low | 1)), 0);
        lo += k * step;
        span = min(step, span - k * step);
    }
    return lo;
}

// Chunks -> rows, 4 rows a workgroup and 64 lines of chunks.
__global__ __launch_bounds__(256) void weights_rows_kernel(const WeightArgs a) {
    __shared__ float2 ml[4][4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, i = lane & 3, p = threadIdx.x >> 2;
    const size_t rows = (size_t)a.tokens * a.hq, row0 = (size_t)blockIdx.x * 4, row = min(row0 + i, rows - 1);
    const int last = (int)(min(row0 + 3, rows - 1) / a.hq), tok = (int)(row / a.hq);
    int n = 0;
    for (int t = (int)(row0 / a.hq); t <= last; ++t) {  // (one token, or a few of few heads)
        const Seq q = seq_of(a, find_seq(a, t, lane));
        if (t == tok && t >= q.row0 && t < q.row0 + q.rows) n = (q.end + a.chunk - 1) / a.chunk;
    }
    float m = -INFINITY, l = 0.0f;
    for (int c = p; c < n; c += 128) {
        const float2 e0 = a.part[(size_t)c * rows + row], e1 = a.part[(size_t)min(c + 64, n - 1) * rows + row];
        add_part(m, l, e0);
        if (c + 64 < n) add_part(m, l, e1);
    }
#pragma unroll
    for (int k = 4; k < 64; k <<= 1) add_part(m, l, make_float2(xor_lane(m, k), xor_lane(l, k)));
    if (lane < 4) ml[wv][i] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= 4 || row0 + i >= rows) return;
    for (int k = 1; k < 4; ++k) add_part(m, l, ml[k][i]);
    a.stat[row] = row_stat(m, l);
}

// The weights of stored x, 4 bytes a row and token: bound by reading them, mostly out of the
// caches that they were just written to (32 sequences, 540K tokens, 8 rows: 35 MB in 15.5 us,
// of which a launch and the statistics are ~5).  A workgroup has one kv head and T tokens, four a lane, whose
// rows its G groups of waves share.  Eight rows' x are on their way while the rows'
// statistics are put together.
constexpr int kSumRows = 64;
template <int T, int G>
__global__ __launch_bounds__(T / 4 * G) void weights_sum_kernel(const WeightArgs a) {
    constexpr int kLanes = T / 4, kThreads = kLanes * G, kGroupRows = G > 4 ? 128 : kSumRows;
    __shared__ float2 st[kGroupRows];
    __shared__ f4 sums[G > 1 ? G - 1 : 1][kLanes];
    const int tid = threadIdx.x;
    const int part = tid % kLanes, grp = __builtin_amdgcn_readfirstlane(tid / kLanes);
    const int blocks = (a.max_kv + T - 1) / T;
    const unsigned b = blockIdx.y * gridDim.x + blockIdx.x;
    const int sh = (int)(b / (unsigned)blocks), blk = (int)(b % (unsigned)blocks);
    const int s = sh / a.g.H, h = sh - s * a.g.H;
    if (s >= a.seqs) return;
    const Seq q = seq_of(a, s);
    if (blk * T >= q.end) return;
    const int C = a.chunk, R = q.rows * a.group, n = (q.end + C - 1) / C, t = blk * T + part * 4;
    const size_t rows = (size_t)a.tokens * a.hq;
    // (x is there up to the end of the last chunk)
    const int at_t = min(t, n * C - 4);
    const auto nat_of = [&](int r) { return query_row(a, q, h, r); };
    constexpr int kDeep = 8;  // rows of a group at a time: grp + G k
    f4 x[kDeep], acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto load = [&](int r0) {
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
            x[k] = *reinterpret_cast<const f4*>(a.logits + (int64_t)nat_of(min(r0 + grp + G * k, R - 1)) * a.logit_stride +
                                                at_t);
    };
    if (R) load(0);
    const int64_t at = (int64_t)sh * a.stride + t;
    // (a row of scores may begin at any float)
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
    const bool four = t + 4 <= q.end;
    f4 before = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.in && grp == 0) {
        if (four)
            before = *reinterpret_cast<const f4u*>(a.in + at);
        else
            for (int k = 0; t + k < q.end; ++k) before[k] = a.in[at + k];
    }
    for (int r0 = 0; r0 < R; r0 += kGroupRows) {
        const int upto = min(kGroupRows, R - r0);
        if (r0) __syncthreads();
        // (16 lanes a row, or fewer for more rows: all of them at once)
        const auto statistics = [&](auto lanes) __attribute__((always_inline)) {
            constexpr int L = decltype(lanes)::value, kRows = kThreads / L;
            const int i = tid % L, p = tid / L;
            float m = -INFINITY, l = 0.0f;
            const size_t nat = nat_of(min(r0 + p, R - 1));
            for (int c = i; c < n; c += 8 * L) {
                float2 e[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = a.part[(size_t)min(c + L * k, n - 1) * rows + nat];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + L * k < n) add_part(m, l, e[k]);
            }
#pragma unroll
            for (int k = 1; k < L; k <<= 1) add_part(m, l, make_float2(xor_lane(m, k), xor_lane(l, k)));
            // (a row that is none: weights of 0)
            if (i == 0 && p < kGroupRows) st[p] = p < upto ? row_stat(m, l) : make_float2(INFINITY, 0.0f);
            for (int r = kRows + tid; r < kGroupRows; r += kThreads) st[r] = make_float2(INFINITY, 0.0f);
        };
        if (upto <= kThreads / 16)
            statistics(std::integral_constant<int, 16>{});
        else
            statistics(std::integral_constant<int, kThreads / kGroupRows>{});
        __syncthreads();
        for (int r = 0; r < upto; r += kDeep * G) {
            if (r0 + r) load(r0 + r);
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const float2 e = st[r + grp + G * k];
#pragma unroll
                for (int w = 0; w < 4; ++w) acc[w] = fmaf(exp2_hw(x[k][w] - e.x), e.y, acc[w]);
            }
        }
    }
    if constexpr (G > 1) {
        if (grp) sums[grp - 1][part] = acc;
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int k = 0; k < G - 1; ++k) acc += sums[k][part];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = a.in ? fmaf(a.decay, before[k], acc[k]) : acc[k];
    if (four)
        *reinterpret_cast<f4u*>(a.out + at) = acc;
    else
        for (int k = 0; t + k < q.end; ++k) a.out[at + k] = acc[k];
}

dim3 grid_of(long long blocks) {
    const unsigned x = (unsigned)std::min<long long>(blocks, 1 << 23);
    return dim3(x, (unsigned)((blocks + x - 1) / x));
}

template <int FMT, int D>
void launch_format(WeightArgs a, hipStream_t stream) {
    constexpr bool kTurned = FMT == kProd || FMT == kMse;
    using B = Blocks<FMT, D>;
    using std::integral_constant;
    const size_t rows = (size_t)a.tokens * a.hq, padded = ((size_t)a.max_kv + 255) / 256 * 256;
    const long long heads = (long long)a.seqs * a.g.H, cus = num_cus();
    const long long per_seq = ((long long)a.tokens * a.group + a.seqs - 1) / a.seqs;  // rows of an average kv head
    // x is stored where that takes less time than K's second reading, its products and a launch
    // more: for up to 64 rows; for little of it; for compressed pages, whose products cost more, as
    // long as each workgroup that adds the rows up has not too many chunks' statistics to go over.
    // Stored / read again in us, 2 kv heads of 128 dims, sequences x tokens, rows:
    //   dense     1 x 2K, 128: 13.9 / 16.9   512: 29.5 / 22.7   1 x 8K, 64: 14.0 / 16.1  128: 18.1 / 17.7
    //             1 x 32K, 64: 27.0 / 24.2   128: 45.8 / 26.8   32 x 8K, 64: 64.1 / 78.0
    //   prod      1 x 2K, 512: 33.8 / 46.6   1 x 8K, 512: 51.1 / 85.6   8 x 4K, 256: 49.0 / 75.6
    //             1 x 32K, 64: 34.0 / 32.2   128: 54.3 / 45.5   32 x 8K, 64: 68.0 / 91
    // Not past 256 MB, which are counted by max_kv for every row: with few rows K's second reading
    // costs far more there, as its blocks are made for many (dense, 8 rows: 32 x 8K tokens 36.5, and
    // one of 120,000 more 72.7, of 131,072 211; 64 x 16,000, 64 heads on 8 523, 64 x 16,500 1,393).
    const size_t stored = rows * padded * 4;
    const bool store = stored <= (size_t(256) << 20) &&
                       (per_seq <= 64 || (kTurned ? a.max_kv <= 16384 : stored <= (size_t(4) << 20)));
    const bool few = store && per_seq <= 16;
    a.chunk = store || kTurned ? 256 : 128;
    a.logit_stride = (int64_t)padded;
    const auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
    const size_t parts = up(((size_t)a.max_kv + a.chunk - 1) / a.chunk * rows * sizeof(float2));
    const size_t second = up(store ? stored : rows * sizeof(float2));
    const size_t turned = kTurned && !few ? up(rows * 4 * D) : 0, scales = kTurned && !few ? up(rows * 4) : 0;
    const float scale = 1.44269504f * inv_sqrt_d(D);
    const WorkspaceTurn turn(stream);
    uint8_t* ws = static_cast<uint8_t*>(Scratch{}.get(stream, parts + second + turned + scales, "attention weights"));
    a.part = reinterpret_cast<float2*>(ws);
    a.logits = reinterpret_cast<float*>(ws + parts);
    a.stat = reinterpret_cast<float2*>(ws + parts);
    a.turned = reinterpret_cast<uint16_t*>(ws + parts + second);
    a.turned_scale = reinterpret_cast<float*>(ws + parts + second + turned);
    if (kTurned && rows && !few) {
        constexpr int per = 256 / (D / 8);
        hipLaunchKernelGGL(turn_queries_kernel<D>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, a.query,
                           a.hq, a.group, (int)rows, const_cast<uint16_t*>(a.turned),
                           const_cast<float*>(a.turned_scale), scale * inv_sqrt_d(D));
        check_launch("attention_weights_turn_kernel");
    }
    const auto chunks_of = [&](int C) { return ((long long)a.max_kv + C - 1) / C; };
    const auto pass = [&](auto wt, auto wr, auto mode, auto block, long long split = 1) {
        constexpr int WT = decltype(wt)::value, WR = decltype(wr)::value, MODE = decltype(mode)::value;
        using S = Shape<FMT, D, WT, WR, MODE, decltype(block)::value>;
        a.row_split = (int)split;
        hipLaunchKernelGGL((weights_kernel<FMT, D, WT, WR, MODE, decltype(block)::value>),
                           grid_of((a.seqs * chunks_of(S::C) + 7) / 8 * 8 * a.g.H * split), dim3(S::kThreads), 0, stream, a,
                           kTurned ? scale * inv_sqrt_d(D) : scale);
        check_launch(MODE == kSum ? "attention_weights_sum_kernel" : "attention_weights_kernel");
    };
    constexpr integral_constant<int, 1> one{};
    constexpr integral_constant<int, 2> two{};  // (waves for tokens x rows: 2 x 2 17.3 + 18.4 us for 256 rows of
                                                // 32K tokens, 4 x 2 22.2 + 19.6, 1 x 4 19.7 + 20.7, 2 x 4 23.7 + 23.3)
    constexpr integral_constant<int, 4> four{};
    // Blocks of few rows or many, and the workgroups that share a chunk's where it has several and
    // the chunks leave compute units without work (prod, 1 x 2K, 512 rows: 132 us without; dense,
    // 1 x 2K, 512 rows: the pass 15.4 us, 7.9 with; 1 x 8K, 128: 6.2, 8.5 with).
    const auto first = [&](auto wt, auto wr, auto mode) {
        const long long work = heads * chunks_of(a.chunk);
        if (per_seq <= B::kSmall)
            pass(wt, wr, mode, integral_constant<int, B::kSmall>{});
        else if (work < (!kTurned ? cus / 4 : store ? 2 * cus : cus))
            pass(wt, wr, mode, integral_constant<int, B::kSmall>{},
                 std::min((per_seq + B::kSmall - 1) / B::kSmall, (4 * cus + work - 1) / work));
        else
            pass(wt, wr, mode, integral_constant<int, B::kLarge>{});
    };
    constexpr integral_constant<int, kStore> storing{};
    constexpr integral_constant<int, kStats> counting{};
    constexpr integral_constant<int, kSum> summing{};
    constexpr integral_constant<int, B::kLarge> large{};
    if (store) {
        if (rows && few)
            pass(four, one, storing, integral_constant<int, B::kFew>{});
        else if (rows)
            first(four, one, storing);
        const long long blocks = chunks_of(1024), smaller = chunks_of(256);
        if (blocks * heads >= 4 * cus)
            hipLaunchKernelGGL((weights_sum_kernel<1024, 1>), grid_of(blocks * heads), dim3(256), 0, stream, a);
        else if (blocks * heads >= cus)  // (32 x 8K tokens, 16 rows: 37.1 us with 256 tokens, 35.2, with 1,024 34.5;
            // 64 rows of compressed pages 53.0, 53.0, 55.1; 32 x 32K, 8 rows: 89.8, 81.2, 78)
            hipLaunchKernelGGL((weights_sum_kernel<512, 2>), grid_of(chunks_of(512) * heads), dim3(256), 0, stream, a);
        else if (per_seq <= 64)  // few workgroups: smaller ones
            hipLaunchKernelGGL((weights_sum_kernel<256, 4>), grid_of(smaller * heads), dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL((weights_sum_kernel<256, 16>), grid_of(smaller * heads), dim3(1024), 0, stream, a);
        check_launch("attention_weights_sum_kernel");
        return;
    }
    if constexpr (kTurned)
        first(four, one, counting);
    else
        first(two, two, counting);
    hipLaunchKernelGGL(weights_rows_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
    check_launch("attention_weights_rows_kernel");
    if constexpr (kTurned)
        pass(four, one, summing, large);
    else if (heads * chunks_of(a.chunk) < cus / 4)  // smaller chunks, whose rows eight waves share: 13.8 us, now 10.9
        pass(one, integral_constant<int, 8>{}, summing, large);
    else
        pass(two, two, summing, large);
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
int weights_entry(const char* name, int fmt, Geom&& geom, const void* query, const uint8_t* pool,
                  const int32_t* tables, int max_blocks, const int32_t* row_start, const int32_t* prefix,
                  int causal, const float* in, float* out, int64_t stride, float decay, int hq, int seqs,
                  int tokens, int max_kv, void* stream) {
    if ((!query && tokens) || !pool || !tables || !row_start || !prefix || !out) return -1;
    try {
        const std::string w = std::string(name) + ": ";
        WeightArgs a{};
        a.g = geom();
        const PageGeom& g = a.g;
        if (g.D != 64 && g.D != 128) throw Error(w + "head_dim must be 64 or 128");
        if (hq <= 0 || hq % g.H || hq > 65535)
            throw Error(w + "num_q_heads must be a multiple of num_kv_heads, at most 65535");
        if (seqs < 0 || tokens < 0) throw Error(w + "num_seqs and num_tokens must be >= 0");
        if (max_blocks <= 0) throw Error(w + "max_blocks_per_seq must be > 0");
        if (max_kv < 0 || max_kv > (1 << 30) || (long long)max_blocks * g.block_size < max_kv)
            throw Error(w + "max_kv_len must be in [0, 2^30] and fit in max_blocks_per_seq pages");
        if (stride < max_kv || stride >= (int64_t(1) << 40))
            throw Error(w + "score_stride must be at least max_kv_len");
        if (!(decay >= 0.0f) || decay > 1.0f) throw Error(w + "decay must be in [0, 1]");
        if ((long long)tokens * hq > (1LL << 25)) throw Error(w + "num_tokens * num_q_heads must be at most 2^25");
        const long long chunks = (max_kv + 127) / 128;
        if (chunks * std::max<long long>((long long)tokens * hq, (long long)seqs * g.H) > (1LL << 30))
            throw Error(w + "too many (row, 128 tokens) or (sequence, kv head, 128 tokens) pairs (2^30)");
        const uint64_t cells = (uint64_t)g.block_size * g.H;
        const auto outside = [&](uint64_t off, uint64_t size) {
            return off > g.page_size || cells * size > g.page_size - off;
        };
        if (outside(g.kc_off, g.code_stride) ||
            (fmt > kBf16 && (outside(g.ks_off, 2) || (fmt == kProd && outside(g.kres_off, 2)))))
            throw Error(w + "layout does not match cfg (a region ends past the page)");
        const uint64_t al = fmt <= kBf16 ? 16 : 2;
        if (!aligned(pool, al) || !aligned(g.page_size | g.kc_off, al) || !aligned(g.ks_off | g.kres_off, 2))
            throw Error(w + (al == 16 ? "page_pool, page size and offsets must be 16-byte aligned"
                                      : "page_pool, page size and offsets must be 2-byte aligned"));
        if (!aligned(query, 16)) throw Error(w + "query must be 16-byte aligned");
        if (!aligned(in, 4) || !aligned(out, 4)) throw Error(w + "scores must be 4-byte aligned");
        if (seqs == 0 || max_kv == 0) return 0;
        a.query = static_cast<const uint16_t*>(query);
        a.pool = pool;
        a.tables = tables;
        a.row_start = row_start;
        a.prefix = prefix;
        a.in = decay == 0.0f ? nullptr : in;
        a.out = out;
        a.stride = stride;
        a.decay = decay;
        a.max_blocks = max_blocks;
        a.hq = hq;
        a.group = hq / g.H;
        while ((1 << a.group_shift) < a.group) ++a.group_shift;
        a.group_mul = (uint32_t)(((1ull << 32) * ((1ull << a.group_shift) - a.group) + a.group - 1) / a.group);
        a.seqs = seqs;
        a.tokens = tokens;
        a.max_kv = max_kv;
        a.causal = causal != 0;
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const auto go = [&](auto f) {
            constexpr int F = decltype(f)::value;
            g.D == 128 ? launch_format<F, 128>(a, st) : launch_format<F, 64>(a, st);
        };
        switch (fmt) {
            case kFp16: go(std::integral_constant<int, kFp16>{}); break;
            case kBf16: go(std::integral_constant<int, kBf16>{}); break;
            case kProd: go(std::integral_constant<int, kProd>{}); break;
            default: go(std::integral_constant<int, kMse>{});
        }
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

extern "C" int tq_launch_dense_attention_weights(
    const void* query, const uint8_t* page_pool, const int32_t* block_tables, int max_blocks_per_seq,
    const int32_t* row_start, const int32_t* prefix_len, int causal, const float* scores_in, float* scores_out,
    int64_t score_stride, float decay, const TQDensePageLayout* layout, const TQConfig* cfg, int dtype,
    int num_q_heads, int num_seqs, int num_tokens, int max_kv_len, void* stream) {
    if (!layout || !cfg) return -1;
    return tq::weights_entry(
        "dense_attention_weights", dtype == TQ_DTYPE_BF16 ? tq::kBf16 : tq::kFp16,
        [&] {
            if (dtype != TQ_DTYPE_FP16 && dtype != TQ_DTYPE_BF16)
                throw tq::Error("dense_attention_weights: dtype must be TQ_DTYPE_FP16 or TQ_DTYPE_BF16");
            return tq::dense_rows(*cfg, *layout);
        },
        query, page_pool, block_tables, max_blocks_per_seq, row_start, prefix_len, causal, scores_in, scores_out,
        score_stride, decay, num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}

extern "C" int tq_launch_turbo_prod_attention_weights(
    const uint16_t* query, const uint8_t* page_pool, const int32_t* block_tables, int max_blocks_per_seq,
    const int32_t* row_start, const int32_t* prefix_len, int causal, const float* scores_in, float* scores_out,
    int64_t score_stride, float decay, const TQTurboProdPageLayout* layout, const TQConfig* cfg,
    int num_q_heads, int num_seqs, int num_tokens, int max_kv_len, void* stream) {
    if (!layout || !cfg) return -1;
    return tq::weights_entry(
        "turbo_prod_attention_weights", tq::kProd, [&] { return tq::prod_geom(*cfg, *layout); }, query, page_pool,
        block_tables, max_blocks_per_seq, row_start, prefix_len, causal, scores_in, scores_out, score_stride, decay,
        num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}

extern "C" int tq_launch_turbo_mse_attention_weights(
    const uint16_t* query, const uint8_t* page_pool, const int32_t* block_tables, int max_blocks_per_seq,
    const int32_t* row_start, const int32_t* prefix_len, int causal, const float* scores_in, float* scores_out,
    int64_t score_stride, float decay, const TQTurbomsePageLayout* layout, const TQConfig* cfg, int num_q_heads,
    int num_seqs, int num_tokens, int max_kv_len, void* stream) {
    if (!layout || !cfg) return -1;
    return tq::weights_entry(
        "turbo_mse_attention_weights", tq::kMse, [&] { return tq::mse_geom(*cfg, *layout); }, query, page_pool,
        block_tables, max_blocks_per_seq, row_start, prefix_len, causal, scores_in, scores_out, score_stride, decay,
        num_q_heads, num_seqs, num_tokens, max_kv_len, stream);
}
