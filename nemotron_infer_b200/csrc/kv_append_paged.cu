// Keys and values of new tokens -> the pages of their sequences, with the rotation by position on the way.
//
//   position of row t of sequence b:  pos = seq_lens[b] - (cu_new[b + 1] - t)
//   K'[t, h] = R(pos) K[t, h],  Q'[t, h] = R(pos) Q[t, h]      R(pos): pairs (x_i, x_j) -> (x_i c - x_j s, x_j c + x_i s)
//   k_cache[page_table[b, pos / P], h, pos % P] = round(K'[t, h] / k_scale),  the same for V without the rotation
//
// Pure streaming: every row is read once and written once (5 KB per token without Q at 8 heads of 128 in bf16, 24.5 KB
// with 40 rotated query heads).  An item is the 16 elements of a head that turn together - two 16-byte vectors, half a
// rotation apart or side by side - so no lane needs another lane's data and every access is 16 bytes wide.  A warp owns
// up to 128 items of ONE token, four per lane with all eight loads issued before the first use; the sequence search, the
// page lookup and the cosine / sine row are then per warp, not per head.
#include "nmt_paged.cuh"

namespace nmt {

constexpr int kAppendWarps = 4;
constexpr int kItemsPerLane = 4;

struct AppendArgs {
    const int32_t* cu;
    const int32_t* seq_lens;
    const int32_t* page_table;
    const __nv_bfloat16 *k, *v, *q;
    __nv_bfloat16* q_out;
    uint8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale, *rope;
    int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, qo_ts, qo_hs;   // token and head strides, elements
    int64_t k_page, v_page;                                      // page strides, elements
    int32_t* err_flag;
    int batch, tokens, kv_heads, q_heads, num_pages, max_pages, page_shift, rope_rows, rot, scale_step, warps_per_token;
};

// (a, b) -> (a c - b s, b c + a s) for the pairs of one item.  INTERLEAVED: a pair is two neighbours of one vector.
template <bool INTERLEAVED>
__device__ __forceinline__ void rotate_item(float (&a)[8], float (&b)[8], const float* __restrict__ row, int half, int first_pair) {
    float c[8], s[8];
    *reinterpret_cast<float4*>(c) = __ldg(reinterpret_cast<const float4*>(row + first_pair));
    *reinterpret_cast<float4*>(c + 4) = __ldg(reinterpret_cast<const float4*>(row + first_pair + 4));
    *reinterpret_cast<float4*>(s) = __ldg(reinterpret_cast<const float4*>(row + half + first_pair));
    *reinterpret_cast<float4*>(s + 4) = __ldg(reinterpret_cast<const float4*>(row + half + first_pair + 4));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float& x = INTERLEAVED ? (i < 4 ? a[2 * i] : b[2 * i - 8]) : a[i];
        float& y = INTERLEAVED ? (i < 4 ? a[2 * i + 1] : b[2 * i - 7]) : b[i];
        const float nx = __fmaf_rn(x, c[i], -__fmul_rn(y, s[i])), ny = __fmaf_rn(y, c[i], __fmul_rn(x, s[i]));
        x = nx;
        y = ny;
    }
}

template <int D, bool E4M3, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendWarps * 32)
kv_append_kernel(const AppendArgs p) {
    constexpr int IPH = D / 16;                                    // items per head
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t gw = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int t = static_cast<int>(gw / p.warps_per_token), part = static_cast<int>(gw % p.warps_per_token);
    if (t >= p.tokens) return;
    int b = t, last = t + 1;
    if (p.cu) {
        b = find_segment(p.cu, p.batch, t);
        if (b < 0) return;
        last = p.cu[b + 1];
        if (t >= last) return;                                     // a row of padding behind the last sequence
    }
    // 64-bit on purpose: lengths and offsets are whatever the caller's device tensors hold
    const int64_t pos = (int64_t)p.seq_lens[b] - ((int64_t)last - t);
    const int64_t pg = pos >> p.page_shift;
    int page = -1;
    if (pos >= 0 && pg < p.max_pages) page = p.page_table[(int64_t)b * p.max_pages + pg];
    if (page < 0 || page >= p.num_pages || (p.rope && pos >= p.rope_rows)) {
        if (p.err_flag && lane == 0) *p.err_flag = 1;
        return;
    }
    const int slot = static_cast<int>(pos) & ((1 << p.page_shift) - 1);
    const int n_kv = p.kv_heads * IPH, n_all = 2 * n_kv + p.q_heads * IPH, half = p.rot >> 1;
    const float* row = p.rope ? p.rope + pos * p.rot : nullptr;
    uint4 va[kItemsPerLane], vb[kItemsPerLane];
    int off_a[kItemsPerLane], off_b[kItemsPerLane];
#pragma unroll
    for (int i = 0; i < kItemsPerLane; ++i) {
        const int item = (part * kItemsPerLane + i) * 32 + lane;
        if (item >= n_all) continue;
        const int kind = item < n_kv ? 0 : item < 2 * n_kv ? 1 : 2;  // K, V, Q
        const int in = item - kind * n_kv, h = in / IPH, j = in % IPH;
        // the two vectors of item j: half a rotation apart while they are rotated (and pairs are not neighbours), else side by side
        const bool split = !INTERLEAVED && kind != 1 && j * 16 < p.rot;
        off_a[i] = split ? j * 8 : j * 16;
        off_b[i] = split ? half + j * 8 : j * 16 + 8;
        const __nv_bfloat16* src = kind == 0 ? p.k + t * p.k_ts + h * p.k_hs : kind == 1 ? p.v + t * p.v_ts + h * p.v_hs : p.q + t * p.q_ts + h * p.q_hs;
        va[i] = ld_stream(reinterpret_cast<const uint4*>(src + off_a[i]));
        vb[i] = ld_stream(reinterpret_cast<const uint4*>(src + off_b[i]));
    }
#pragma unroll
    for (int i = 0; i < kItemsPerLane; ++i) {
        const int item = (part * kItemsPerLane + i) * 32 + lane;
        if (item >= n_all) continue;
        const int kind = item < n_kv ? 0 : item < 2 * n_kv ? 1 : 2;
        const int in = item - kind * n_kv, h = in / IPH, j = in % IPH;
        const bool turn = kind != 1 && j * 16 < p.rot;
        float a[8], c[8];
        if (turn || E4M3) {
            unpack8(va[i], a);
            unpack8(vb[i], c);
        }
        if (turn) {
            rotate_item<INTERLEAVED>(a, c, row, half, j * 8);
            if (!E4M3 || kind == 2) { va[i] = pack8(a); vb[i] = pack8(c); }
        }
        if (kind == 2) {
            __nv_bfloat16* dst = p.q_out + t * p.qo_ts + h * p.qo_hs;
            st_stream(reinterpret_cast<uint4*>(dst + off_a[i]), va[i]);
            st_stream(reinterpret_cast<uint4*>(dst + off_b[i]), vb[i]);
            continue;
        }
        uint8_t* base = kind == 0 ? p.k_cache : p.v_cache;
        const int64_t at = (int64_t)page * (kind == 0 ? p.k_page : p.v_page) + ((int64_t)(h << p.page_shift) + slot) * D;
        if (!E4M3) {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(base) + at;
            *reinterpret_cast<uint4*>(dst + off_a[i]) = va[i];
            *reinterpret_cast<uint4*>(dst + off_b[i]) = vb[i];
        } else {
            const float* sc = kind == 0 ? p.k_scale : p.v_scale;
            const float s = sc ? __ldg(sc + h * p.scale_step) : 1.f;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                w[e] = e4m3x2_rn(__fdiv_rn(a[4 * e], s), __fdiv_rn(a[4 * e + 1], s)) |
                       (e4m3x2_rn(__fdiv_rn(a[4 * e + 2], s), __fdiv_rn(a[4 * e + 3], s)) << 16);
                w[2 + e] = e4m3x2_rn(__fdiv_rn(c[4 * e], s), __fdiv_rn(c[4 * e + 1], s)) |
                           (e4m3x2_rn(__fdiv_rn(c[4 * e + 2], s), __fdiv_rn(c[4 * e + 3], s)) << 16);
            }
            *reinterpret_cast<uint2*>(base + at + off_a[i]) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(base + at + off_b[i]) = make_uint2(w[2], w[3]);
        }
    }
    pdl_trigger();
}

}  // namespace nmt

extern "C" {

int nmt_kv_append_paged_bf16(const nmt_paged_cache* c, const int32_t* cu_new, int64_t tokens, const void* k, int64_t k_ts, int64_t k_hs,
                             const void* v, int64_t v_ts, int64_t v_hs, const float* rope, int64_t rope_rows, int64_t rot_dim, int interleaved,
                             const void* q, int64_t q_ts, int64_t q_hs, int64_t q_heads, void* q_out, int64_t qo_ts, int64_t qo_hs,
                             int32_t* err_flag, void* stream) {
    using namespace nmt;
    int st = check_paged_cache(c);
    if (st != NMT_OK) return st;
    if (tokens < 0 || tokens > 0x7fffffff || (!cu_new && tokens != c->batch)) return NMT_ERR_SHAPE;
    if (!q) q_heads = 0;
    if (q && (!q_out || !rope)) return NMT_ERR_NULL;
    if (q && (q_heads <= 0 || q_heads > 65535)) return NMT_ERR_SHAPE;
    if (rope && (rope_rows <= 0 || rope_rows > 0x7fffffff || rot_dim <= 0 || (rot_dim & 15) || rot_dim > c->head_dim)) return NMT_ERR_SHAPE;
    if (tokens == 0 || c->batch == 0) return NMT_OK;
    if (!c->k || !c->v || !c->page_table || !c->seq_lens) return NMT_ERR_NULL;
    if ((st = check_view(k, tokens, k_ts, c->kv_heads, k_hs)) != NMT_OK || (st = check_view(v, tokens, v_ts, c->kv_heads, v_hs)) != NMT_OK) return st;
    if (q && ((st = check_view(q, tokens, q_ts, q_heads, q_hs)) != NMT_OK || (st = check_view(q_out, tokens, qo_ts, q_heads, qo_hs)) != NMT_OK)) return st;
    if (!aligned4(cu_new) || !aligned4(err_flag) || !aligned16(rope)) return NMT_ERR_ALIGN;
    AppendArgs p;
    p.cu = cu_new; p.seq_lens = c->seq_lens; p.page_table = c->page_table;
    p.k = static_cast<const __nv_bfloat16*>(k); p.v = static_cast<const __nv_bfloat16*>(v); p.q = static_cast<const __nv_bfloat16*>(q);
    p.q_out = static_cast<__nv_bfloat16*>(q_out);
    p.k_cache = static_cast<uint8_t*>(c->k); p.v_cache = static_cast<uint8_t*>(c->v);
    p.k_scale = c->k_scale; p.v_scale = c->v_scale; p.rope = rope;
    p.k_ts = k_ts; p.k_hs = k_hs; p.v_ts = v_ts; p.v_hs = v_hs; p.q_ts = q_ts; p.q_hs = q_hs; p.qo_ts = qo_ts; p.qo_hs = qo_hs;
    p.k_page = c->k_page_stride; p.v_page = c->v_page_stride;
    p.err_flag = err_flag;
    p.batch = static_cast<int>(c->batch); p.tokens = static_cast<int>(tokens); p.kv_heads = static_cast<int>(c->kv_heads);
    p.q_heads = static_cast<int>(q_heads); p.num_pages = static_cast<int>(c->num_pages); p.max_pages = static_cast<int>(c->max_pages);
    p.page_shift = log2_of(c->page_size); p.rope_rows = static_cast<int>(rope_rows); p.rot = rope ? static_cast<int>(rot_dim) : 0;
    p.scale_step = c->scale_count > 1 ? 1 : 0;
    const int64_t items = (2 * c->kv_heads + q_heads) * (c->head_dim / 16);
    p.warps_per_token = static_cast<int>((items + 32 * kItemsPerLane - 1) / (32 * kItemsPerLane));
    const int64_t ctas = (tokens * p.warps_per_token + kAppendWarps - 1) / kAppendWarps;
    if (ctas > 0x7fffffff) return NMT_ERR_UNSUPPORTED;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    const bool e4m3 = c->dtype == NMT_CACHE_E4M3;
#define NMT_APPEND(D, E, I) launch_kernel(kv_append_kernel<D, E, I>, static_cast<int>(ctas), kAppendWarps * 32, 0, cs, p)
#define NMT_APPEND_D(D)                                                                  \
    do {                                                                                 \
        if (e4m3) { if (interleaved) NMT_APPEND(D, true, true); else NMT_APPEND(D, true, false); } \
        else { if (interleaved) NMT_APPEND(D, false, true); else NMT_APPEND(D, false, false); }    \
    } while (0)
    if (c->head_dim == 128) NMT_APPEND_D(128); else NMT_APPEND_D(64);
#undef NMT_APPEND_D
#undef NMT_APPEND
    return finish_launch(1);
}

}  // extern "C"
