// Attention of whole prompts on the 5th-generation tensor cores, causal or not, grouped heads, packed sequences.
//
//   out[i, h] = sum_j p_ij v[j, g],   p_ij = softmax_j(scale q[i, h] . k[j, g]),   j <= i + (m - n) when causal
//
// One pass over the keys with a running maximum M and sum L per query row:  P = 2^(c S - M),  L += sum P,  O += P V,
// O *= 2^(M_old - M_new) when M moves (c = scale log2 e).  M is allowed to lag behind the true maximum by a factor of 2^8
// - any M gives the same O / L - so after a row's first tiles O is hardly ever rescaled.
//
// A work item is two query tiles, 128 rows of a head each, that share every K / V tile of 128 keys: two heads of a group on the
// same rows, or the next rows (all of them, where there is one head per group).  One CTA per SM, 16 warps with fixed roles:
//   warps 0-3, 4-7   softmax of query tile 0 / 1: a thread owns a row.  Reads S from tensor memory, writes P (bf16) over it
//   warps 8-11       epilogue: O / L -> bf16 -> global memory, while the other warps are at the next item already
//   warp 12          issues the MMAs (one lane)
//   warp 13          producer: finds the next item, publishes it, and copies its Q, K, V into shared memory (tensor maps)
// S_t = Q_t K^T: tcgen05.mma 128 x 128 x 16 from shared memory (both operands rows of 128 bytes, 128-byte swizzle) into
// tensor memory.  O_t += P_t V: A comes from tensor memory, where P_t lies over S_t's first 64 columns, B is V as it lies
// in memory (keys x head_dim, so MN-major).  Columns 0-127 S_0 / P_0, 128-255 S_1 / P_1, 256-383 O_0, 384-511 O_1: all 512.
// The MMAs of the two tiles alternate, PV_0 S_0' PV_1 S_1', so the tensor core works on one tile while the softmax warps are
// on the other.  MMAs run in the order they are issued, and a commit covers all of them before it: "S_t is ready" also says
// that the previous PV_t is done, which is what a rescale of O_t needs, so no other signal is exchanged per tile.
#include "nmt_paged.cuh"
#include "nmt_tensormap.cuh"
#include "nmt_tma.cuh"

namespace nmt {

NMT_DEFINE_TIMEOUT_READER();

constexpr int kPfThreads = 512;
constexpr int kPfTile = 128;                                       // rows of a query tile, keys of a K / V tile
constexpr int kSoftmaxRegs = 200, kEpilogueRegs = 56, kOtherRegs = 56;    // 2 x 200 + 56 + 56 = 512 = 4 x the launch's 128
constexpr float kLag = 8.f;                                        // log2 of how far M may lag

// Cutting an item's keys into pieces, when there are fewer items than SMs' worth of work (a few new queries over a long prefix).
constexpr int kPfMinPiece = 8;                                     // K / V tiles of a piece, at least
constexpr int kPfSlack = 4;                                        // an item this much over the average is left whole
constexpr int kPfPieces = 2 * kSmCount;                            // pieces there can be (see pieces())
constexpr int kPfSplitItems = 4 * kSmCount;                        // with more items than this nothing is cut

template <int D>
struct PfShape {
    static constexpr int kTileBytes = kPfTile * D * 2;             // Q tile, K tile or V tile
    static constexpr int kStages = D == 128 ? 5 : 10;              // 160 KB of K / V tiles
    static constexpr int kHalves = D / 64;                         // 64-column halves of 128-byte rows
    static constexpr size_t kSmem = 1024 + (size_t)(2 + kStages) * kTileBytes;
};

struct PrefillArgs {
    __nv_bfloat16* out;
    float* part_o;                                 // pieces: [kPfPieces][2][128][D] sums of weights times values; NULL: nothing is cut
    float2* part_ml;                               // [kPfPieces][2][128]: maximum (log 2 units) and sum of the weights
    const __nv_bfloat16 *q, *k, *v;
    const int32_t *cu_q, *cu_k;
    int64_t o_ts, o_hs, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    float scale_log2;
    int batch, q_tokens, kv_tokens, kv_heads, group, causal, out32;   // out32: rows of out are 32-byte aligned
};

struct PfItem {
    int kv_row;                                    // first key of the sequence in k and v
    int kv_len, kv_head;
    // per query tile: first row in q and out, valid rows (1 .. 128), keys that row 0 sees before clamping (row r sees limit + r
    // when causal), head, K / V tiles.  n[0] < 0: no more items; n[1] == 0: one query tile only.  n[0] <= n[1] otherwise.
    int q_row[2], rows[2], limit[2], head[2], n[2];
    int first;                                     // first K / V tile: 0 unless this is a piece of a cut item
    int slot;                                      // where a piece leaves its result; < 0: a whole item, written to out
};

// Shared-memory matrix descriptors, as two words so that a step along an operand is one 32-bit addition.  High word: 1024
// bytes between groups of 8 rows (bits 32-45, in 16 bytes), version 1 (bit 46), 128-byte swizzle (2 at bit 61).  Low word:
// address / 16, and at bit 16 the leading offset / 16.  K-major in rows of 128 bytes: not used, 1.  MN-major (V: rows are k,
// 64 columns of n each): a whole half of the tile, 16 KB, to the next 64 columns.
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mnmajor(uint32_t addr) { return (addr >> 4) | (1024u << 16); }
// D fp32 (bits 4-5), A and B bf16 (bits 7-9, 10-12), B MN-major at bit 16, N / 8 at bits 17-22, M / 16 at bits 24-28.
template <int N, bool B_MN>
__host__ __device__ constexpr uint32_t idesc_bf16() {
    return (1u << 4) | (1u << 7) | (1u << 10) | (B_MN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(kPfTile >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile("{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %4, 0; mov.b64 da, {%1, %5}; mov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "r"(kDescHigh) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile("{ .reg .pred p; .reg .b64 db; setp.ne.b32 p, %4, 0; mov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p; }"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "r"(kDescHigh) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ uint32_t warp_uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define NMT_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define NMT_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
// 32 columns of this warp's 32 lanes: thread = lane, register = column.
__device__ __forceinline__ void tm_ld32(uint32_t* r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
                 "%26,%27,%28,%29,%30,%31}, [%32];"
                 : NMT_R8(r, 0), NMT_R8(r, 8), NMT_R8(r, 16), NMT_R8(r, 24) : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t* r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : NMT_R8(r, 0), NMT_R8(r, 8) : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::NMT_W8(r, 0), NMT_W8(r, 8), "r"(addr) : "memory");
}
__device__ __forceinline__ void tma_rows(uint32_t smem_dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger of three; a NaN among them is kept.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x on the FMA pipe, two at a time, for -inf < x < 128.  x is kept at or above -127, where the result is an exact zero (and
// between there and -126 anything below 2^-126).  x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves it in the low bits of the sum), f in [-1/2, 1/2], and 2^f by a polynomial of
// degree 4 with constant term 1, fitted for the least relative error (minimax, by linear programming): 2.9e-6 = 2^-18.4,
// against the 2^-8 of the rounding to bf16 that follows.  n goes into the exponent by an integer addition.
__device__ __forceinline__ float2 ex2_fma(const float2& x) {
    const float2 magic = make_float2(12582912.f, 12582912.f);
    const float2 xc = make_float2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
    const float2 t = __fadd2_rn(xc, magic);
    const float2 f = __fadd2_rn(xc, __ffma2_rn(t, make_float2(-1.f, -1.f), magic));
    float2 y = __ffma2_rn(f, make_float2(0.009582576341927052f, 0.009582576341927052f), make_float2(0.05590682849287987f, 0.05590682849287987f));
    y = __ffma2_rn(y, f, make_float2(0.24024106562137604f, 0.24024106562137604f));
    y = __ffma2_rn(y, f, make_float2(0.6931241154670715f, 0.6931241154670715f));
    y = __ffma2_rn(y, f, make_float2(1.f, 1.f));
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}
// The weights of one row of a tile from its scores: w = 2^(s c - mc), added to the row sum in fp32, rounded to bf16 and
// written over the scores in tensor memory, half a tile at a time so that the product with V can start on the first half.
// PLAIN: every exponential on the special-function unit, exact zeros and NaN included (masked, infinite or NaN scores).
// Otherwise kFmaPairs of every 8 pairs go to the FMA pipe: the special-function unit gives 16 results per cycle and SM,
// which for 2 x 128 x 128 weights is as long as the four products that the tensor core does meanwhile.
constexpr int kFmaPairs = 2;
template <bool PLAIN>
__device__ __forceinline__ void weights(const float (&s)[kPfTile], const float2& c2, float mc, float2& l2, uint32_t p_addr, int lane, uint64_t* half_bar,
                                        uint64_t* full_bar) {
    const float2 nm2 = make_float2(-mc, -mc);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const float2 x = __ffma2_rn(make_float2(s[64 * h + 2 * e], s[64 * h + 2 * e + 1]), c2, nm2);
            const bool fma = !PLAIN && (e * kFmaPairs) % 8 < kFmaPairs;
            const float2 y = fma ? ex2_fma(x) : make_float2(pf_ex2(x.x), pf_ex2(x.y));
            sum[e & 1] = __fadd2_rn(sum[e & 1], y);
            pk[e] = pack2(y);
            if (e == 15) tm_st16(p_addr + 32 * h, pk);
        }
        tm_st16(p_addr + 32 * h + 16, pk + 16);
        tm_wait_st();
        tm_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(h == 0 ? half_bar : full_bar);
    }
    l2 = __fadd2_rn(l2, __fadd2_rn(sum[0], sum[1]));
}
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct PfBarriers {
    uint64_t item_full[2], item_empty[2], q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2], l_full[2];
    uint64_t kv_full[10], kv_empty[10], v_raw, taken;
};

// A lane-0 wait broadcast to the warp: everybody agrees on whether it ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_now(bar, parity)); }

// The query tiles of a sequence and kv head - blocks of 128 rows, and for each the heads of the group - are numbered block by
// block, heads first, and an item is two neighbours: mostly two heads on the same rows, which see the same keys.  A short
// prompt then fills both tiles of an item (with 256 rows of one head per item, 64 prompts of 128 tokens took 69 us instead of 55).
// Items are handed out by their number of K / V tiles, most first, so that the last ones to start are short; among
// equals sequence by sequence, kv heads fastest.  The lengths are only known on the device; a warp counts as it goes - the
// numbers it is given only grow, so it keeps its place.
struct PfSequence {
    int q0, n, k0, m;                              // first query row, query rows, first key, keys
    __device__ __forceinline__ PfSequence(const PrefillArgs& p, int b) : q0(0), n(p.q_tokens), k0(0), m(p.kv_tokens) {
        if (!p.cu_q) return;
        const int32_t* cu_k = p.cu_k ? p.cu_k : p.cu_q;
        q0 = min(max(p.cu_q[b], 0), p.q_tokens);
        n = min(max(p.cu_q[b + 1], q0), p.q_tokens) - q0;
        k0 = min(max(cu_k[b], 0), p.kv_tokens);
        m = min(max(cu_k[b + 1], k0), p.kv_tokens) - k0;
    }
    __device__ __forceinline__ int tiles(const PrefillArgs& p) const { return (n + kPfTile - 1) / kPfTile * p.group; }
    __device__ __forceinline__ int items(const PrefillArgs& p) const { return (tiles(p) + 1) / 2; }
    // Items (the last ones) with at least `cost` K / V tiles; an item that sees nothing counts as one tile.
    __device__ __forceinline__ int items_from(const PrefillArgs& p, int cost) const {
        const int all = items(p), keys = (cost - 1) * kPfTile;     // such an item's last row sees more than `keys`
        if (cost <= 1 || all == 0) return all;
        if (m <= keys) return 0;
        if (!p.causal) return all;
        const int short_of = keys - (m - n);                       // the last row of block x sees m - n + min(n, 128 (x + 1)) keys
        const int block = short_of < 0 ? 0 : min(short_of / kPfTile, (n - 1) / kPfTile);
        return all - block * p.group / 2;                          // items whose second tile is in that block or a later one
    }
    // K / V tiles of the longest item, and of the shortest.
    __device__ __forceinline__ int longest() const { return n > 0 ? max(1, (m + kPfTile - 1) / kPfTile) : 0; }
    __device__ __forceinline__ int shortest(const PrefillArgs& p) const {
        if (!p.causal || n == 0) return longest();
        const int block = p.group == 1 && n > kPfTile ? 1 : 0;     // of the first item's second query tile
        return max(1, (min(m, m - n + min(n, (block + 1) * kPfTile)) + kPfTile - 1) / kPfTile);
    }
    // K / V tiles of all items together: the sum over c of items_from(c).
    __device__ __forceinline__ int64_t work(const PrefillArgs& p) const {
        const int64_t all = items(p), most = (m + kPfTile - 1) / kPfTile;
        if (!p.causal || most <= 1) return all * max(most, (int64_t)1);
        // items_from(c) = all - floor(k G / 2) with k = max(c - 1 - e, 0), e = ceil((m - n) / 128), for c = 2 .. most
        const int64_t e = m >= n ? (m - n + kPfTile - 1) / kPfTile : -((n - m) / kPfTile), g = p.group;
        auto sum = [&](int64_t x) {                                // of floor(k G / 2), k = 0 .. x
            return x <= 0 ? (int64_t)0 : (g * (x * (x + 1) / 2) - ((g & 1) ? (x + 1) / 2 : 0)) / 2;
        };
        return all * most - (sum(most - 1 - e) - sum(e < 0 ? -e : 0));
    }
};
struct PfOrder {
    int cost, base, count, chunk, before;          // cost now handed out, pieces of higher cost, items of this one; place among the sequences
    int below;                                     // the next lower cost that some item has
    int share;                                     // K / V tiles that would be every SM's equal part, or more than any item has

    // Pieces of an item with c K / V tiles.  Only items of more than `share` are cut, into fewer than 2 c / share pieces, and all
    // items together have at most share * kSmCount tiles: at most kPfPieces pieces, the first in the order.
    __device__ __forceinline__ int pieces(int c) const { return c <= share + kPfSlack ? 1 : (c + share - 1) / share; }

    __device__ __forceinline__ void seat(const PrefillArgs& p, int c) {
        cost = c;
        chunk = before = 0;
        int mine = 0, next = 0;
        if (cost > 0)
            for (int b = threadIdx.x & 31; b < p.batch; b += 32) {
                const PfSequence q(p, b);
                mine += q.items_from(p, cost) - q.items_from(p, cost + 1);
                const int lower = min(cost - 1, q.longest());
                if (lower >= q.shortest(p)) next = max(next, lower);
            }
        count = __reduce_add_sync(0xffffffffu, mine);
        below = __reduce_max_sync(0xffffffffu, next);
    }
    __device__ __forceinline__ void start(const PrefillArgs& p) {
        int most = 0;
        int64_t all = 0;
        for (int b = threadIdx.x & 31; b < p.batch; b += 32) {
            const PfSequence q(p, b);
            most = max(most, q.longest());
            all += q.work(p);
        }
        share = 0x3fffffff;
        if (p.part_o) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
            share = static_cast<int>(min(max((all * p.kv_heads + kSmCount - 1) / kSmCount, (int64_t)kPfMinPiece), (int64_t)0x3fffffff));
        }
        base = 0;
        seat(p, __reduce_max_sync(0xffffffffu, most));
    }
    __device__ __forceinline__ int piece_len() const { return (cost + pieces(cost) - 1) / pieces(cost); }
    // The which-th item that is cut, as its first piece.  False: there is no such item.
    __device__ __forceinline__ bool find_cut(const PrefillArgs& p, int which, PfItem& it) {
        int items = 0;                                             // of higher cost
        while (cost > 0 && pieces(cost) > 1 && which >= items + count * p.kv_heads) {
            items += count * p.kv_heads;
            base += count * p.kv_heads * pieces(cost);
            seat(p, below);
        }
        return cost > 0 && pieces(cost) > 1 && find(p, base + (which - items) * pieces(cost), it);
    }
    // The piece or item with this number.  False: there is none.
    __device__ __forceinline__ bool find(const PrefillArgs& p, int index, PfItem& it) {
        const int lane = threadIdx.x & 31;
        while (cost > 0 && index >= base + count * p.kv_heads * pieces(cost)) {
            base += count * p.kv_heads * pieces(cost);
            seat(p, below);
        }
        if (cost <= 0) return false;
        const int cut = pieces(cost), piece = (index - base) % cut, which = (index - base) / cut;
        const int rank = which / p.kv_heads;
        it.kv_head = which % p.kv_heads;
        // the sequence whose share of this cost holds `rank`
        int mine, upto;
        for (;;) {
            mine = 0;
            if (chunk + lane < p.batch) {
                const PfSequence q(p, chunk + lane);
                mine = q.items_from(p, cost) - q.items_from(p, cost + 1);
            }
            upto = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += up;
            }
            const int sum = __shfl_sync(0xffffffffu, upto, 31);
            if (rank < before + sum || chunk + 32 >= p.batch) break;
            before += sum;
            chunk += 32;
        }
        const uint32_t holds = __ballot_sync(0xffffffffu, rank - before < upto && rank - before >= upto - mine);
        const int src = max(__ffs(holds) - 1, 0);
        const PfSequence q(p, min(chunk + src, p.batch - 1));
        const int in_share = rank - before - __shfl_sync(0xffffffffu, upto - mine, src);
        const int item = q.items(p) - q.items_from(p, cost) + in_share, tiles = q.tiles(p);
        it.kv_row = q.k0;
        it.kv_len = q.m;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int x = min(2 * item + t, tiles - 1), first = x / p.group * kPfTile;
            it.head[t] = it.kv_head * p.group + x % p.group;
            it.q_row[t] = q.q0 + first;
            it.rows[t] = min(kPfTile, q.n - first);
            it.limit[t] = p.causal ? first + 1 + (q.m - q.n) : q.m;
            const int sees = p.causal ? min(q.m, it.limit[t] + it.rows[t] - 1) : q.m;
            it.n[t] = 2 * item + t < tiles ? max(1, (sees + kPfTile - 1) / kPfTile) : 0;
        }
        const int len = piece_len();
        it.first = piece * len;
        it.slot = cut > 1 ? index : -1;
        if (cut > 1)
#pragma unroll
            for (int t = 0; t < 2; ++t) it.n[t] = min(max(it.n[t] - it.first, 0), len);
        return holds != 0;
    }
};

// The grid has a CTA for every item, but only one per SM fits: a running CTA takes over the work of one that has not started
// yet (cluster launch control), so the items go to whoever is free.  The answer is 16 bytes in shared memory.
__device__ __forceinline__ void ask_for_cta(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int cta_taken(const void* answer) {     // its index, or -1: none was left
    uint32_t ok, x;
    asm volatile("{ .reg .pred p; .reg .b128 h; ld.shared.b128 h, [%2];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h; selp.u32 %0, 1, 0, p; mov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h; }"
                 : "=r"(ok), "=r"(x) : "r"(smem_u32(answer)) : "memory");
    return ok ? static_cast<int>(x) : -1;
}

// One row again, by a warp on the CUDA cores, over the keys it sees and no others.  A tile product multiplies the hidden
// keys' values by weights of zero, which is wrong where such a value is an infinity or a NaN (0 x NaN is NaN): the epilogue
// sends a row here when its sum is finite and its output is not.  Without such values no call comes here.
template <int D>
__device__ __forceinline__ void redo_row(const PrefillArgs& p, int q_row, int head, int kv_row, int sees) {
    constexpr int W = D / 64;                                      // words (pairs of elements) per lane
    const int lane = threadIdx.x & 31;
    const __nv_bfloat16* qp = p.q + (int64_t)q_row * p.q_ts + (int64_t)head * p.q_hs;
    const __nv_bfloat16* kp = p.k + (int64_t)kv_row * p.k_ts + (int64_t)(head / p.group) * p.k_hs;
    const __nv_bfloat16* vp = p.v + (int64_t)kv_row * p.v_ts + (int64_t)(head / p.group) * p.v_hs;
    __nv_bfloat16* dst = p.out + (int64_t)q_row * p.o_ts + (int64_t)head * p.o_hs;
    float2 q[W], o[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        q[i] = unpack2(*reinterpret_cast<const uint32_t*>(qp + i * 64 + lane * 2));
        o[i] = make_float2(0.f, 0.f);
    }
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int j = 0; j < sees; ++j) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float2 k = unpack2(*reinterpret_cast<const uint32_t*>(kp + j * p.k_ts + i * 64 + lane * 2));
            dot = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, dot));
        }
        const float s = warp_sum(dot) * p.scale_log2, to = fmaxf(m, s);
        const float f = m == -INFINITY ? 0.f : exp2f(m - to), w = to == -INFINITY ? 0.f : exp2f(s - to);
        const bool moved = to > m;                                 // a factor of one is left out: 0 x inf is no part of the formula
        m = to;
        l = (moved ? l * f : l) + w;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float2 v = unpack2(*reinterpret_cast<const uint32_t*>(vp + j * p.v_ts + i * 64 + lane * 2));
            o[i].x = fmaf(w, v.x, moved ? o[i].x * f : o[i].x);
            o[i].y = fmaf(w, v.y, moved ? o[i].y * f : o[i].y);
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) *reinterpret_cast<uint32_t*>(dst + i * 64 + lane * 2) = pack_bf16x2(o[i].x / l, o[i].y / l);
}

template <int D>
__global__ void __launch_bounds__(kPfThreads, 1)
sdpa_prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const PrefillArgs p) {
    using Shape = PfShape<D>;
    constexpr int ST = Shape::kStages;
    extern __shared__ __align__(1024) uint8_t smem_p[];
    __shared__ PfBarriers bar;
    __shared__ PfItem s_item[2];
    __shared__ __align__(16) uint4 s_answer;
    __shared__ float s_l[2][kPfTile];
    __shared__ uint32_t s_tmem;
    const int lane = threadIdx.x & 31, warp = static_cast<int>(warp_uniform(threadIdx.x >> 5));
    const uint32_t q_smem = (smem_u32(smem_p) + 1023u) & ~1023u, ring = q_smem + 2 * Shape::kTileBytes;
    if (threadIdx.x == 0) {
        prefetch_map(&qmap);
        prefetch_map(&kmap);
        prefetch_map(&vmap);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.item_full[i], 1);
            mbar_init(&bar.item_empty[i], 13);                     // warps 0-12
            mbar_init(&bar.q_full[i], 1);
            mbar_init(&bar.q_empty[i], 1);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_half[i], 4);
            mbar_init(&bar.p_full[i], 4);
            mbar_init(&bar.o_full[i], 1);
            mbar_init(&bar.o_empty[i], 4);
            mbar_init(&bar.l_full[i], 4);
        }
        mbar_init(&bar.v_raw, 1);
        mbar_init(&bar.taken, 1);
        for (int i = 0; i < ST; ++i) { mbar_init(&bar.kv_full[i], 1); mbar_init(&bar.kv_empty[i], 1); }
        mbar_init_fence();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    const uint32_t tmem = warp_uniform(*reinterpret_cast<volatile uint32_t*>(&s_tmem));
    pdl_wait();

    // Every role runs the same loop over the published items.  A wait that runs out (counted, nmt_tma.cuh) ends the role's
    // loop; the other roles' waits then run out too, nothing is left waiting for good.
    auto next_item = [&](int k, PfItem& it) {
        if (!warp_wait(&bar.item_full[k & 1], static_cast<uint32_t>(k >> 1) & 1u)) return false;
        it = s_item[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.item_empty[k & 1]);
        return it.n[0] >= 0;
    };

    if (warp < 8) {
        // ---------------- softmax ----------------
        regs_up<kSoftmaxRegs>();
        const int t = warp >> 2, wq = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
        const uint32_t s_addr = tmem + lanes + t * kPfTile, o_addr = tmem + lanes + 256 + t * kPfTile;
        const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
        uint32_t s_uses = 0, o_uses = 0;
        PfItem it;
        for (int k = 0; next_item(k, it); ++k) {
            const int tiles = t == 0 ? it.n[0] : it.n[1];
            if (tiles == 0) continue;
            const int sees = p.causal ? min(it.kv_len, (t == 0 ? it.limit[0] : it.limit[1]) + wq * 32 + lane) : it.kv_len;
            float m = -INFINITY;                                   // M / c
            float2 l2 = make_float2(0.f, 0.f);
            bool ok = true;
            for (int j = 0; j < tiles; ++j) {
                ok = warp_wait(&bar.s_full[t], s_uses & 1u);
                if (!ok) break;
                ++s_uses;
                tm_fence_after();
                float s[kPfTile];
                float top4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) tm_ld32(reinterpret_cast<uint32_t*>(s) + 32 * c, s_addr + 32 * c);
                tm_wait_ld();
                const int left = sees - (it.first + j) * kPfTile;
                const bool masked = __any_sync(0xffffffffu, left < kPfTile);
                if (masked) {
#pragma unroll
                    for (int c = 0; c < kPfTile; ++c) s[c] = c < left ? s[c] : -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top4[c] = s[32 * c];
#pragma unroll
                    for (int e = 1; e < 31; e += 2) top4[c] = max3_nan(top4[c], s[32 * c + e], s[32 * c + e + 1]);
                }
                const float top = max3_nan(max3_nan(top4[0], s[31], s[63]), max3_nan(top4[1], s[95], s[127]), max3_nan(top4[2], top4[2], top4[3]));
                // M moves only when it has to: the first tile, or a maximum more than 2^8 above it
                const bool move = (top - m) * p.scale_log2 > kLag || (m == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float to = move ? top : m;
                    const float f = move ? pf_ex2((m - to) * p.scale_log2) : 1.f;       // m == -inf: 0
                    l2.x *= f;
                    l2.y *= f;
                    if (j > 0) {
                        uint32_t o[16];
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {          // rare, and 128 scores are live: few registers, no unrolling
                            tm_ld16(o, o_addr + c);
                            tm_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tm_st16(o_addr + c, o);
                        }
                    }
                    m = to;
                }
                const float mc = m == -INFINITY ? 0.f : m * p.scale_log2;
                // a maximum that is not finite: a NaN or infinite score, or a row that sees nothing here
                if (masked || __any_sync(0xffffffffu, !(fabsf(top) < INFINITY))) weights<true>(s, c2, mc, l2, s_addr, lane, &bar.p_half[t], &bar.p_full[t]);
                else weights<false>(s, c2, mc, l2, s_addr, lane, &bar.p_half[t], &bar.p_full[t]);
            }
            if (!ok) break;
            if (o_uses > 0 && !warp_wait(&bar.o_empty[t], (o_uses - 1) & 1u)) break;    // the last item's L has been read
            ++o_uses;
            s_l[t][wq * 32 + lane] = l2.x + l2.y;
            if (it.slot >= 0) p.part_ml[((size_t)it.slot * 2 + t) * kPfTile + wq * 32 + lane] = make_float2(m * p.scale_log2, l2.x + l2.y);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.l_full[t]);
        }
    } else if (warp < 12) {
        // ---------------- epilogue ----------------
        regs_down<kEpilogueRegs>();
        const int wq = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
        uint32_t uses[2] = {0, 0};
        PfItem it;
        bool ok = true;
        for (int k = 0; ok && next_item(k, it); ++k) {
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {                          // loops that are not unrolled: short items are bound by the instructions they run through once
                if ((t == 0 ? it.n[0] : it.n[1]) == 0 || !ok) continue;
                const uint32_t phase = (t == 0 ? uses[0]++ : uses[1]++) & 1u;
                ok = warp_wait(&bar.l_full[t], phase) && warp_wait(&bar.o_full[t], phase);
                if (!ok) continue;
                tm_fence_after();
                const int r = wq * 32 + lane, q_row = t == 0 ? it.q_row[0] : it.q_row[1], head = t == 0 ? it.head[0] : it.head[1];
                const int limit = t == 0 ? it.limit[0] : it.limit[1];
                const bool valid = r < (t == 0 ? it.rows[0] : it.rows[1]);
                const float l = s_l[t][r];
                const int sees = p.causal ? min(it.kv_len, limit + r) : it.kv_len;
                const bool none = sees <= 0 || l == 0.f;           // nothing to average: zeros, whatever the product holds
                const float2 inv2 = make_float2(1.f / l, 1.f / l);
                __nv_bfloat16* dst = p.out + (int64_t)(q_row + r) * p.o_ts + (int64_t)head * p.o_hs;
                float* part = p.part_o + (((size_t)max(it.slot, 0) * 2 + t) * kPfTile + r) * D;
                uint32_t o_addr = tmem + lanes + 256 + t * kPfTile;
                float2 odd2 = make_float2(0.f, 0.f);               // 0 x (a value that is not finite) is NaN
                auto put = [&](const uint32_t (&o)[16]) {          // 16 columns
                    if (it.slot >= 0) {                            // a piece: as it is, for the join
                        if (valid) {
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(part), NMT_W8(o, 0) : "memory");
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(part + 8), NMT_W8(o, 8) : "memory");
                        }
                        part += 16;
                        return;
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 f = __fmul2_rn(make_float2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])), inv2);
                        odd2 = __ffma2_rn(f, make_float2(0.f, 0.f), odd2);
                        w[e] = none ? 0u : pack2(f);
                    }
                    if (valid) {
                        if (p.out32) {
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), NMT_W8(w, 0) : "memory");
                        } else {
                            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                    dst += 16;
                };
                uint32_t oa[16], ob[16];                           // one is on its way while the other is stored
                tm_ld16(oa, o_addr);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    tm_wait_ld();
                    tm_ld16(ob, o_addr + 16);
                    put(oa);
                    tm_wait_ld();
                    o_addr += 32;
                    if (c + 32 < D) {
                        tm_ld16(oa, o_addr);
                    } else {                                       // O and L are in registers: the next item may have them
                        tm_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.o_empty[t]);
                    }
                    put(ob);
                }
                const bool odd = !none && valid && it.slot < 0 && odd2.x + odd2.y != 0.f;
                for (uint32_t redo = __ballot_sync(0xffffffffu, odd && l < INFINITY); redo; redo &= redo - 1) {
                    const int rr = wq * 32 + __ffs(redo) - 1;
                    redo_row<D>(p, q_row + rr, head, it.kv_row, p.causal ? min(it.kv_len, limit + rr) : it.kv_len);
                }
            }
        }
    } else {
        regs_down<kOtherRegs>();
        if (warp == 12) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t kIdS = idesc_bf16<kPfTile, false>(), kIdO = idesc_bf16<D, true>();
            uint32_t q_uses[2] = {0, 0}, p_uses[2] = {0, 0}, o_uses[2] = {0, 0}, kv = 0;      // kv: tiles taken from the ring
            PfItem it;
            bool ok = true;
            auto stage_of = [&](uint32_t i) { return static_cast<int>(i % ST); };
            auto wait_kv = [&](uint32_t i) { return warp_wait(&bar.kv_full[stage_of(i)], (i / ST) & 1u); };
            auto scores = [&](int t, uint32_t ki) {                // S_t = Q_t K^T
                const uint32_t qa = warp_uniform(desc_kmajor(q_smem + t * Shape::kTileBytes));
                const uint32_t ka = warp_uniform(desc_kmajor(ring + stage_of(ki) * Shape::kTileBytes));
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4);
                        mma_ss(tmem + t * kPfTile, qa + off, ka + off, kIdS, kk > 0);
                    }
                    mma_commit(&bar.s_full[t]);
                }
            };
            for (int k = 0; ok && next_item(k, it); ++k) {
                const int n_max = max(it.n[0], it.n[1]);
                ok = wait_kv(kv);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (it.n[t] == 0 || !ok) continue;
                    ok = warp_wait(&bar.q_full[t], q_uses[t]++ & 1u);
                    if (!ok) continue;
                    tm_fence_after();
                    scores(t, kv);
                    if (it.n[t] == 1 && elect_one()) mma_commit(&bar.q_empty[t]);
                }
                if (ok && elect_one()) mma_commit(&bar.kv_empty[stage_of(kv)]);
                for (int j = 0; j < n_max && ok; ++j) {
                    const uint32_t vi = kv + 2 * j + 1, ki = vi + 1;
                    ok = wait_kv(vi) && (j + 1 >= n_max || wait_kv(ki));
                    if (!ok) break;
                    const uint32_t vd = warp_uniform(desc_mnmajor(ring + stage_of(vi) * Shape::kTileBytes));
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok) continue;
                        if (j < it.n[t]) {
                            if (j == 0 && o_uses[t] > 0) ok = warp_wait(&bar.o_empty[t], (o_uses[t] - 1) & 1u);
                            // the weights come in two halves of 64 keys
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                ok = ok && warp_wait(h == 0 ? &bar.p_half[t] : &bar.p_full[t], p_uses[t] & 1u);
                                if (!ok) continue;
                                tm_fence_after();
                                if (elect_one()) {
#pragma unroll
                                    for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                                        mma_ts(tmem + 256 + t * kPfTile, tmem + t * kPfTile + kk * 8, vd + kk * (2048 >> 4), kIdO, j > 0 || kk > 0);
                                    if (h == 1 && j == it.n[t] - 1) mma_commit(&bar.o_full[t]);
                                }
                            }
                            ++p_uses[t];
                            if (!ok) continue;
                            if (j == it.n[t] - 1) ++o_uses[t];
                        }
                        if (j + 1 < it.n[t]) {
                            scores(t, ki);
                            if (j + 2 == it.n[t] && elect_one()) mma_commit(&bar.q_empty[t]);
                        }
                    }
                    if (ok && elect_one()) {
                        mma_commit(&bar.kv_empty[stage_of(vi)]);
                        if (j + 1 < n_max) mma_commit(&bar.kv_empty[stage_of(ki)]);
                    }
                    __syncwarp();
                }
                kv += 2 * n_max;
            }
        } else if (warp == 13) {
            // ---------------- producer ----------------
            uint32_t q_uses[2] = {0, 0}, kv = 0, v_raws = 0;
            PfOrder order;
            PfItem it;
            bool ok = true;
            auto load = [&](const CUtensorMap* map, int head, int row, uint32_t dst, uint64_t* full) {
                if (elect_one()) {
                    mbar_arrive_expect_tx(full, Shape::kTileBytes);
#pragma unroll
                    for (int h = 0; h < Shape::kHalves; ++h) tma_rows(dst + h * 16384, map, h * 64, head, row, full);
                }
            };
            auto publish = [&](int k) {
                if (k >= 2) ok = warp_wait(&bar.item_empty[k & 1], static_cast<uint32_t>((k >> 1) - 1) & 1u);
                if (ok && lane == 0) {
                    s_item[k & 1] = it;
                    mbar_arrive(&bar.item_full[k & 1]);
                }
                __syncwarp();
            };
            int k = 0, index = blockIdx.x, asked = 0;
            order.start(p);
            auto ask = [&] {
                if (elect_one()) {
                    mbar_arrive_expect_tx(&bar.taken, 16);
                    ask_for_cta(&s_answer, &bar.taken);
                }
                ++asked;
            };
            auto answer = [&] {
                if (!warp_wait(&bar.taken, static_cast<uint32_t>(asked - 1) & 1u)) return false;
                index = cta_taken(&s_answer);
                fence_proxy_async_smem();                          // this read before the next answer is written
                __syncwarp();
                return true;
            };
            while (ok && index >= 0) {
                if (!order.find(p, index, it)) {                   // past the real number: take these CTAs out of the way too
                    ask();
                    ok = answer();
                    continue;
                }
                publish(k++);
                const int n_max = max(it.n[0], it.n[1]);
                auto load_q = [&](int t) {
                    if (it.n[t] == 0 || !ok) return;
                    if (q_uses[t] > 0) ok = warp_wait(&bar.q_empty[t], (q_uses[t] - 1) & 1u);
                    if (!ok) return;
                    ++q_uses[t];
                    load(&qmap, it.head[t], it.q_row[t], q_smem + t * Shape::kTileBytes, &bar.q_full[t]);
                };
                if (ok) load_q(0);
                for (int i = 0; i < 2 * n_max && ok; ++i, ++kv) {
                    // the next item is asked for when this one's last tiles go out, not earlier: whoever is free shall have it
                    if (i == max(0, 2 * n_max - 4)) ask();
                    const int st = static_cast<int>(kv % ST);
                    if (kv >= ST) ok = warp_wait(&bar.kv_empty[st], (kv / ST - 1) & 1u);
                    if (!ok) break;
                    const uint32_t dst = ring + st * Shape::kTileBytes;
                    const int tile = it.first + (i >> 1), valid = it.kv_len - tile * kPfTile;
                    if ((i & 1) && valid < kPfTile) {
                        // Keys past the sequence's end belong to another one or to nobody, and 0 x NaN is NaN: their rows of V
                        // are cleared before anybody is told that the tile is there.
                        load(&vmap, it.kv_head, it.kv_row + tile * kPfTile, dst, &bar.v_raw);
                        ok = warp_wait(&bar.v_raw, v_raws++ & 1u);
                        if (!ok) break;
                        const int from = max(valid, 0);
                        for (int x = lane; x < (kPfTile - from) * 8 * Shape::kHalves; x += 32) {
                            const int r = from + x / (8 * Shape::kHalves), y = x % (8 * Shape::kHalves);
                            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst + (y >> 3) * 16384 + r * 128 + (y & 7) * 16), "r"(0u) : "memory");
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.kv_full[st]);
                        __syncwarp();
                    } else {
                        load(i & 1 ? &vmap : &kmap, it.kv_head, it.kv_row + tile * kPfTile, dst, &bar.kv_full[st]);
                    }
                    if (i == 0) load_q(1);
                }
                ok = ok && answer();
            }
            it.n[0] = -1;
            if (ok) publish(k);
            // no copy may still be under way when the CTA gives up its shared memory
            if (lane == 0) {
                for (uint32_t i = kv > ST ? kv - ST : 0; i < kv; ++i) mbar_wait(&bar.kv_full[i % ST], (i / ST) & 1u);
                for (int t = 0; t < 2; ++t)
                    if (q_uses[t] > 0) mbar_wait(&bar.q_full[t], (q_uses[t] - 1) & 1u);
                if (v_raws > 0) mbar_wait(&bar.v_raw, (v_raws - 1) & 1u);
                if (asked > 0) mbar_wait(&bar.taken, static_cast<uint32_t>(asked - 1) & 1u);
            }
        }
    }
    tm_fence_before();
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    pdl_trigger();
}

// Joins the pieces of the items that were cut: CTA (i, t, quarter) takes 32 rows of query tile t of the i-th such item; a warp
// takes a row at a time, a lane D / 32 columns.  The order of items is worked out again, which is shorter than passing it
// on would be.
constexpr int kPfJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kPfJoinWarps * 32)
sdpa_prefill_join_kernel(const PrefillArgs p) {
    constexpr int W = D / 64;
    __shared__ PfItem s_it;
    __shared__ int s_cut, s_len;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.y;
    pdl_wait();
    if (warp == 0) {
        PfOrder order;
        PfItem it;
        order.start(p);
        const bool have = order.find_cut(p, blockIdx.x, it);
        if (lane == 0) {
            s_cut = have ? order.pieces(order.cost) : 0;
            s_len = have ? order.piece_len() : 0;
            s_it = it;
        }
    }
    __syncthreads();
    const PfItem& it = s_it;
    const int cut = s_cut, len = s_len;
    if (cut > 0 && it.n[t] > 0) {
        for (int r = blockIdx.z * 32 + warp; r < min(it.rows[t], static_cast<int>(blockIdx.z) * 32 + 32); r += kPfJoinWarps) {
            const int sees = p.causal ? min(it.kv_len, it.limit[t] + r) : it.kv_len;
            // pieces past the last key that the row sees hold nothing of it (and may not have looked at this tile at all)
            const int n = min(cut, max(1, (sees + len * kPfTile - 1) / (len * kPfTile)));
            auto at = [&](int i) { return ((size_t)(it.slot + i) * 2 + t) * kPfTile + r; };
            float top = -INFINITY;
#pragma unroll 4
            for (int i = 0; i < n; ++i) top = fmaxf(top, p.part_ml[at(i)].x);
            float sum = 0.f;
            float2 acc[W];
#pragma unroll
            for (int e = 0; e < W; ++e) acc[e] = make_float2(0.f, 0.f);
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const float2 ml = p.part_ml[at(i)];
                if (ml.y == 0.f) continue;                         // sees nothing there: whatever its products hold
                const float w = pf_ex2(ml.x - (top == -INFINITY ? 0.f : top));
                sum = fmaf(w, ml.y, sum);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float2 o = *reinterpret_cast<const float2*>(p.part_o + at(i) * D + e * 64 + lane * 2);
                    acc[e].x = fmaf(w, o.x, acc[e].x);
                    acc[e].y = fmaf(w, o.y, acc[e].y);
                }
            }
            const bool none = sees <= 0 || sum == 0.f;
            bool odd = false;
            __nv_bfloat16* dst = p.out + (int64_t)(it.q_row[t] + r) * p.o_ts + (int64_t)it.head[t] * p.o_hs;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float x = none ? 0.f : acc[e].x / sum, y = none ? 0.f : acc[e].y / sum;
                odd |= !(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY);
                *reinterpret_cast<uint32_t*>(dst + e * 64 + lane * 2) = pack_bf16x2(x, y);
            }
            if (__any_sync(0xffffffffu, odd) && sum < INFINITY) redo_row<D>(p, it.q_row[t] + r, it.head[t], it.kv_row, sees);
        }
    }
    pdl_trigger();
}

template <int D>
static void launch_prefill(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const PrefillArgs& p, int items, cudaStream_t st) {
    auto kern = sdpa_prefill_kernel<D>;
    static std::atomic<uint64_t> allowed{0};
    allow_smem(kern, PfShape<D>::kSmem, allowed);
    launch_kernel(kern, items + (p.part_o ? kPfPieces : 0), kPfThreads, PfShape<D>::kSmem, st, qm, km, vm, p);
    if (p.part_o) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(kSmCount, 2, kPfTile / 32);             // a cut item has more than an SM's equal part: fewer than kSmCount of them
        cfg.blockDim = dim3(kPfJoinWarps * 32);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 1 : 0;
        cudaLaunchKernelEx(&cfg, sdpa_prefill_join_kernel<D>, p);
    }
}

// Items: two query tiles (128 rows of a head) of a sequence and kv head each.  As many as the batch can have (every sequence
// may end in a partly filled block and an odd tile); CTAs past the real number find nothing to do.
static int64_t prefill_items(int64_t batch, int64_t q_tokens, int64_t heads, int64_t kv_heads) {
    const int64_t full = (q_tokens + kPfTile - 1) / kPfTile, blocks = q_tokens < full + batch - 1 ? q_tokens : full + batch - 1;
    return (blocks * (heads / kv_heads) + (blocks < batch ? blocks : batch)) / 2 * kv_heads;
}
// Whether some item can be worth cutting, from what the host knows: few items, and keys for at least two pieces.  One
// sequence is known well enough to tell that its longest item is no more than an SM's equal part.
static bool prefill_may_cut(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads) {
    const int64_t most = (kv_tokens + kPfTile - 1) / kPfTile, items = prefill_items(batch, q_tokens, heads, kv_heads);
    if (items > kPfSplitItems || most <= kPfMinPiece + kPfSlack) return false;
    return batch > 1 || (most - kPfSlack) * kSmCount > items * (2 * kv_tokens - q_tokens) / (2 * kPfTile);
}

}  // namespace nmt

extern "C" {

int64_t nmt_sdpa_prefill_workspace_bytes(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
    using namespace nmt;
    if (batch <= 0 || q_tokens <= 0 || kv_tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || heads % kv_heads) return 0;
    return prefill_may_cut(batch, q_tokens, kv_tokens, heads, kv_heads) ? (int64_t)kPfPieces * 2 * kPfTile * (head_dim * 4 + 8) : 0;
}

int nmt_sdpa_prefill_bf16(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                          int64_t v_hs, void* out, int64_t o_ts, int64_t o_hs, const int32_t* cu_q, const int32_t* cu_k, int64_t batch,
                          int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                          void* workspace, void* stream) {
    using namespace nmt;
    if (batch < 0 || q_tokens < 0 || kv_tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || !(scale > 0.f) || !(scale < INFINITY))
        return NMT_ERR_SHAPE;
    if ((!cu_q && (batch != 1 || cu_k))) return NMT_ERR_SHAPE;
    if (head_dim != 64 && head_dim != 128) return NMT_ERR_UNSUPPORTED;
    if (q_tokens > 0x3fffffff || kv_tokens > 0x3fffffff || batch > 0x3fffffff || heads > 65535) return NMT_ERR_UNSUPPORTED;
    const int64_t items = prefill_items(batch, q_tokens, heads, kv_heads);
    if (items > 0x3fffffff) return NMT_ERR_UNSUPPORTED;
    if (q_tokens == 0 || batch == 0) return NMT_OK;
    int st;
    if ((st = check_view(q, q_tokens, q_ts, heads, q_hs)) != NMT_OK || (st = check_view(out, q_tokens, o_ts, heads, o_hs)) != NMT_OK) return st;
    if (kv_tokens > 0 && ((st = check_view(k, kv_tokens, k_ts, kv_heads, k_hs)) != NMT_OK || (st = check_view(v, kv_tokens, v_ts, kv_heads, v_hs)) != NMT_OK))
        return st;
    if (!aligned4(cu_q) || !aligned4(cu_k) || (reinterpret_cast<uintptr_t>(workspace) & 31u)) return NMT_ERR_ALIGN;
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return NMT_ERR_UNSUPPORTED;
    // Without keys there is nothing to describe (and nothing that is read counts): any valid row will do.
    const bool none = kv_tokens == 0;
    struct { const void* p; int64_t tokens, ts, heads, hs; } views[3] = {{q, q_tokens, q_ts, heads, q_hs},
                                                                       {none ? q : k, none ? 1 : kv_tokens, k_ts, none ? 1 : kv_heads, k_hs},
                                                                       {none ? q : v, none ? 1 : kv_tokens, v_ts, none ? 1 : kv_heads, v_hs}};
    CUtensorMap maps[3];
    for (int i = 0; i < 3; ++i) {
        const auto& w = views[i];
        const int64_t hs = w.heads > 1 ? w.hs : head_dim, ts = w.tokens > 1 ? w.ts : head_dim * w.heads;
        if ((w.heads > 1 && hs < 1) || (w.tokens > 1 && ts < 1)) return NMT_ERR_UNSUPPORTED;       // a broadcast view
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(w.heads), static_cast<cuuint64_t>(w.tokens)};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(hs * 2), static_cast<cuuint64_t>(ts * 2)};
        const cuuint32_t box[3] = {64, 1, kPfTile}, ones[3] = {1, 1, 1};
        if (encode(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(w.p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return NMT_ERR_UNSUPPORTED;
    }
    PrefillArgs p;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.q = static_cast<const __nv_bfloat16*>(q); p.k = static_cast<const __nv_bfloat16*>(k); p.v = static_cast<const __nv_bfloat16*>(v);
    p.cu_q = cu_q; p.cu_k = cu_k; p.o_ts = o_ts; p.o_hs = o_hs;
    p.q_ts = q_ts; p.q_hs = q_hs; p.k_ts = k_ts; p.k_hs = k_hs; p.v_ts = v_ts; p.v_hs = v_hs;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.batch = static_cast<int>(batch); p.q_tokens = static_cast<int>(q_tokens); p.kv_tokens = static_cast<int>(kv_tokens);
    p.kv_heads = static_cast<int>(kv_heads); p.group = static_cast<int>(heads / kv_heads); p.causal = causal != 0;
    p.out32 = (reinterpret_cast<uintptr_t>(out) & 31u) == 0 && (q_tokens == 1 || o_ts % 16 == 0) && (heads == 1 || o_hs % 16 == 0);
    const bool cut = workspace && prefill_may_cut(batch, q_tokens, kv_tokens, heads, kv_heads);
    p.part_o = cut ? static_cast<float*>(workspace) : nullptr;
    p.part_ml = cut ? reinterpret_cast<float2*>(p.part_o + (size_t)kPfPieces * 2 * kPfTile * head_dim) : nullptr;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (head_dim == 128) launch_prefill<128>(maps[0], maps[1], maps[2], p, static_cast<int>(items), cs);
    else launch_prefill<64>(maps[0], maps[1], maps[2], p, static_cast<int>(items), cs);
    return finish_launch(cut ? 2 : 1);
}

}  // extern "C"
