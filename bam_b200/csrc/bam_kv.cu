/*
 * bam_kv.cu -- a key/value cache kept in the pages of an array: append (norm of each head and position rotation on
 * the way), gather, and attention of one new token per sequence.
 *
 * The reference has no counterpart: its consumers are graph and array kernels.  The pages are reached the way those
 * reach theirs -- look up, pin, read or write, unpin; a page that is not in the cache is fetched from the store
 * through the NVMe queues by the same launch -- so the rows of a cache larger than HBM need no other handling.
 */
#include <cuda_runtime.h>

#include <cstring>

#include "bam_kv.cuh"

using namespace bam;

/* ====================================================================================== */
/* append                                                                                  */
/* ====================================================================================== */

#define KV_MAX_LANE_TOKENS 32u

struct kv_rope_d_t {
    const int64_t* positions;
    const float *cos, *sin;
    uint64_t n_positions;
    int64_t stride;
    uint32_t rotary_dim;         /* 0: no rotation                                             */
    uint32_t style;              /* BAM_KV_ROPE_HALF / BAM_KV_ROPE_PAIRS                       */
};

/* One row of a head: G lanes (a power of two, at least head_dim / 8) hold eight elements each.  All lanes of the
 * warp call it.  y = x * rsqrt(mean(x^2) + eps) * w, then the rotation; everything in 32 bits, rounded once. */
template <class T>
BAM_DEV uint4 kv_transform(uint4 raw, uint32_t c, uint32_t G, uint32_t head_dim, const uint16_t* norm, float eps,
                           const kv_rope_d_t& rope, int64_t pos)
{
    if (!norm && rope.rotary_dim == 0) return raw;
    float x[8];
    {
        const uint32_t w[4] = { raw.x, raw.y, raw.z, raw.w };
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = kv_type<T>::unpack(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    const bool in_row = c * 8 < head_dim;
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i];
        if (!in_row) ss = 0.f;
        for (uint32_t o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss / (float)head_dim + eps);
        if (in_row) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = x[i] * inv * kv_type<T>::to_f(norm[c * 8 + i]);
        }
    }
    const uint32_t half = rope.rotary_dim >> 1;
    if (rope.rotary_dim) {
        if (rope.style == BAM_KV_ROPE_HALF) {
            /* the other element of a pair lies rotary_dim / 2 away: half / 8 lanes (rotary_dim is a multiple of 16) */
            const bool low = c * 8 < half, turned = c * 8 < rope.rotary_dim;
            const uint32_t other = turned ? (low ? c + half / 8 : c - half / 8) : c;
            const uint32_t src = ((threadIdx.x & 31u) & ~(G - 1u)) + other;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = __shfl_sync(0xffffffffu, x[i], src);
            if (turned) {
                const uint32_t e = low ? c * 8 : c * 8 - half;
                const float* cs = rope.cos + pos * rope.stride + e;
                const float* sn = rope.sin + pos * rope.stride + e;
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = low ? x[i] * __ldg(cs + i) - p[i] * __ldg(sn + i) : x[i] * __ldg(cs + i) + p[i] * __ldg(sn + i);
            }
        } else if (c * 8 < rope.rotary_dim) {
            const float* cs = rope.cos + pos * rope.stride + c * 4;
            const float* sn = rope.sin + pos * rope.stride + c * 4;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float a = x[2 * i], b = x[2 * i + 1], cc = __ldg(cs + i), ss = __ldg(sn + i);
                x[2 * i] = a * cc - b * ss;
                x[2 * i + 1] = b * cc + a * ss;
            }
        }
    }
    return make_uint4(kv_type<T>::pack(x[0], x[1]), kv_type<T>::pack(x[2], x[3]), kv_type<T>::pack(x[4], x[5]), kv_type<T>::pack(x[6], x[7]));
}

/* Pins the pages of up to 32 rows, one per lane, and hands the rows of every page that could be pinned to `rows`,
 * which all lanes call together with the mask of lanes whose page is there; pages are released before the warp asks
 * again for the others, so that a warp never holds one page while it waits for another.  Returns false after a failure. */
template <class Rows>
BAM_DEV bool kv_with_pages(const kv_layout_d_t& L, bool want, uint64_t page, bool write, uint32_t queue, Rows rows)
{
    const uint32_t full = 0xffffffffu, lane = lane_id();
    bool pending = want;
    spin_t sp;
    while (__any_sync(full, pending)) {
        const uint32_t slot = kv_pin_warp(L, pending, page, write, queue);
        const bool got = pending && slot <= BAM_SLOT_MAX;
        const bool failed = __any_sync(full, pending && slot == BAM_SLOT_ERR);
        const uint32_t m = __ballot_sync(full, got);
        if (m && !failed) rows(m, got ? L.r.get_cache_page_addr(slot) : 0);
        if (write) __threadfence();
        __syncwarp();
        /* one release per page: the lowest of the lanes that share it gives all their counts back */
        const uint32_t same = __match_any_sync(full, got ? slot : ~lane);
        if (got && lane == (uint32_t)(__ffs(same) - 1)) L.r.release_page(slot, __popc(same));
        if (failed) return false;
        if (got) pending = false;
        if (m == 0u && __any_sync(full, sp.expired(L.r.cache.status, BAM_AT_FIND_SLOT, page))) return false;
    }
    return true;
}

template <class T>
struct KvAppendWork {
    static constexpr int threads = BAM_THREADS, min_blocks = 2;
    static constexpr uint32_t smem = BAM_FUSED_SMEM;
    kv_layout_d_t L;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh;      /* element strides of token and head */
    uint64_t n_tokens;
    uint32_t n_q_heads, lanes_per_row, tokens_per_item;
    uint32_t vec;                                                  /* bit 0: q, 1: k, 2: v, 3: q_out lie on 16-byte boundaries */
    const int64_t* slots;
    kv_rope_d_t rope;
    const uint16_t *q_norm, *k_norm;
    float eps;

    /* the position of a token, or -1 after the error has been recorded */
    BAM_DEV int64_t position(uint64_t t, bool padded) const
    {
        if (rope.rotary_dim == 0) return 0;
        const int64_t p = rope.positions[t];
        if (p >= 0 && (uint64_t)p < rope.n_positions) return p;
        if (padded) return p < 0 ? 0 : (int64_t)rope.n_positions - 1;
        L.bad_index((uint64_t)p);
        return -1;
    }

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        const uint32_t lane = threadIdx.x & 31u;
        const uint64_t warp = ((uint64_t)vb * blockDim.x + threadIdx.x) >> 5, nwarps = ((uint64_t)nvb * blockDim.x) >> 5;
        const uint32_t G = lanes_per_row, rows = 32u / G, c = lane & (G - 1u), grp = lane / G;
        const bool in_row = c < L.chunks;
        if (status_bad(L.r.cache.status)) return;
        /* keys and values: an item is tokens_per_item tokens of one head */
        const uint64_t groups = (n_tokens + tokens_per_item - 1) / tokens_per_item;
        for (uint64_t it = warp; it < groups * L.n_kv_heads; it += nwarps) {
            const uint32_t h = (uint32_t)(it % L.n_kv_heads);
            const uint64_t t0 = it / L.n_kv_heads * tokens_per_item;
            const uint64_t t = t0 + lane;
            int64_t slot = -1, pos = 0;
            if (lane < tokens_per_item && t < n_tokens) {
                slot = slots[t];
                if (slot >= 0 && (uint64_t)slot >= L.n_blocks * L.block_tokens) {
                    L.bad_index((uint64_t)slot);
                    slot = -1;
                }
                if (slot >= 0) pos = position(t, false);
                if (pos < 0) slot = -1;
            }
            const uint32_t row = slot >= 0 ? (uint32_t)((uint64_t)slot % L.block_tokens) : 0;
            const uint64_t page = slot >= 0 ? L.page_of((uint64_t)slot / L.block_tokens, h) : 0;
            const bool ok = kv_with_pages(L, slot >= 0, page, true, (uint32_t)warp, [&](uint32_t m, uint64_t addr) {
                for (uint32_t i = 0; i < tokens_per_item; i += rows) {
                    const uint32_t src = (i + grp) & 31u;
                    if (!((m >> i) & ((rows == 32u) ? 0xffffffffu : (1u << rows) - 1u))) continue;
                    const bool act = in_row && i + grp < tokens_per_item && ((m >> src) & 1u);
                    const uint64_t base = __shfl_sync(0xffffffffu, addr, src);
                    const uint32_t rr = __shfl_sync(0xffffffffu, row, src);
                    const int64_t pp = __shfl_sync(0xffffffffu, pos, src);
                    uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
                    if (act) {
                        kk = kv_load8(k + (int64_t)(t0 + src) * k_st + h * k_sh + c * 8, vec & 2u);
                        vv = kv_load8(v + (int64_t)(t0 + src) * v_st + h * v_sh + c * 8, vec & 4u);
                    }
                    kk = kv_transform<T>(kk, c, G, L.head_dim, k_norm, eps, rope, pp);
                    if (act) {
                        uint8_t* p = reinterpret_cast<uint8_t*>(base) + rr * L.row_bytes() + L.swizzle(rr, c) * 16u;
                        *reinterpret_cast<uint4*>(p) = kk;
                        *reinterpret_cast<uint4*>(p + L.v_offset()) = vv;
                    }
                }
            });
            if (!ok) return;
        }
        /* queries */
        if (!q) return;
        const uint64_t n_rows = n_tokens * n_q_heads;
        for (uint64_t r0 = warp * rows; r0 < n_rows; r0 += nwarps * rows) {
            const uint64_t rr = r0 + grp;
            const bool act = in_row && rr < n_rows;
            const uint64_t t = act ? rr / n_q_heads : 0;
            const uint32_t h = act ? (uint32_t)(rr % n_q_heads) : 0;
            uint4 x = make_uint4(0, 0, 0, 0);
            int64_t pos = 0;
            if (act) {
                x = kv_load8(q + (int64_t)t * q_st + h * q_sh + c * 8, vec & 1u);
                pos = position(t, slots[t] < 0);
                if (pos < 0) pos = 0;
            }
            x = kv_transform<T>(x, c, G, L.head_dim, q_norm, eps, rope, pos);
            if (act) kv_store8(q_out + (int64_t)t * qo_st + h * qo_sh + c * 8, x, vec & 8u);
        }
    }
};

/* ====================================================================================== */
/* gather                                                                                  */
/* ====================================================================================== */

struct KvGatherWork {
    static constexpr int threads = BAM_THREADS, min_blocks = 2;
    static constexpr uint32_t smem = BAM_FUSED_SMEM;
    kv_layout_d_t L;
    uint16_t *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;
    uint64_t n_tokens;
    uint32_t lanes_per_row, tokens_per_item;
    uint32_t vec;
    const int64_t* slots;

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        const uint32_t lane = threadIdx.x & 31u;
        const uint64_t warp = ((uint64_t)vb * blockDim.x + threadIdx.x) >> 5, nwarps = ((uint64_t)nvb * blockDim.x) >> 5;
        const uint32_t G = lanes_per_row, rows = 32u / G, c = lane & (G - 1u), grp = lane / G;
        const bool in_row = c < L.chunks;
        if (status_bad(L.r.cache.status)) return;
        const uint64_t groups = (n_tokens + tokens_per_item - 1) / tokens_per_item;
        for (uint64_t it = warp; it < groups * L.n_kv_heads; it += nwarps) {
            const uint32_t h = (uint32_t)(it % L.n_kv_heads);
            const uint64_t t0 = it / L.n_kv_heads * tokens_per_item;
            const uint64_t t = t0 + lane;
            const bool mine = lane < tokens_per_item && t < n_tokens;
            int64_t slot = mine ? slots[t] : -1;
            if (slot >= 0 && (uint64_t)slot >= L.n_blocks * L.block_tokens) {
                L.bad_index((uint64_t)slot);
                slot = -1;
            }
            const uint32_t row = slot >= 0 ? (uint32_t)((uint64_t)slot % L.block_tokens) : 0;
            const uint64_t page = slot >= 0 ? L.page_of((uint64_t)slot / L.block_tokens, h) : 0;
            auto copy = [&](uint32_t m, uint64_t addr) {
                for (uint32_t i = 0; i < tokens_per_item; i += rows) {
                    const uint32_t src = (i + grp) & 31u;
                    const bool act = in_row && i + grp < tokens_per_item && ((m >> src) & 1u);
                    const uint64_t base = __shfl_sync(0xffffffffu, addr, src);
                    const uint32_t rr = __shfl_sync(0xffffffffu, row, src);
                    if (act) {
                        uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
                        if (base) {
                            /* past L1: a slot can hold another page now than earlier in this launch */
                            const uint8_t* p = reinterpret_cast<const uint8_t*>(base) + rr * L.row_bytes() + L.swizzle(rr, c) * 16u;
                            kk = ld_cg_v4(p);
                            vv = ld_cg_v4(p + L.v_offset());
                        }
                        kv_store8(k + (int64_t)(t0 + src) * k_st + h * k_sh + c * 8, kk, vec & 1u);
                        kv_store8(v + (int64_t)(t0 + src) * v_st + h * v_sh + c * 8, vv, vec & 2u);
                    }
                }
            };
            const uint32_t padded = __ballot_sync(0xffffffffu, mine && slot < 0);
            if (padded) copy(padded, 0);
            if (!kv_with_pages(L, slot >= 0, page, false, (uint32_t)warp, copy)) return;
        }
    }
};

/* ====================================================================================== */
/* host side                                                                               */
/* ====================================================================================== */

namespace {

int kv_layout(bam_array* a, const bam_kv_layout_t* l, kv_layout_d_t* L)
{
    if (!a || !l) return BAM_EINVAL;
    if (a->n_ranges != 1 || a->h_range.page_start_offset) return BAM_EINVAL;       /* pages are addressed directly */
    if (l->dtype != BAM_KV_BF16 && l->dtype != BAM_KV_FP16) return BAM_EINVAL;
    if (l->head_dim < 16 || l->head_dim > 256 || l->head_dim % 16) return BAM_EINVAL;
    if (l->n_kv_heads == 0 || l->n_kv_heads > 65536 || l->n_blocks == 0 || l->n_blocks > 0x7fffffffull) return BAM_EINVAL;
    if (l->block_tokens == 0 || l->block_tokens % 16 || (uint64_t)l->block_tokens * l->head_dim * 4 > a->pc->d.page_size) return BAM_EINVAL;
    const uint64_t pages = l->n_blocks * l->n_kv_heads;
    if (l->first_page > a->h_range.page_count || pages > a->h_range.page_count - l->first_page) return BAM_ERANGE;
    memset(L, 0, sizeof *L);
    L->r = a->h_range;
    L->first_page = l->first_page; L->n_blocks = l->n_blocks;
    L->head_dim = l->head_dim; L->n_kv_heads = l->n_kv_heads; L->block_tokens = l->block_tokens;
    L->chunks = l->head_dim / 8;
    switch (L->chunks % 8) {
    case 0: L->swz_shift = 0; L->swz_mask = 7; break;
    case 4: L->swz_shift = 1; L->swz_mask = 3; break;
    default: L->swz_shift = 2; L->swz_mask = 1; break;           /* 2 or 6: head_dim is a multiple of 16 */
    }
    return BAM_OK;
}

uint32_t lanes_of_row(uint32_t chunks) { uint32_t g = 1; while (g < chunks) g <<= 1; return g; }

bool on_16(const void* p, int64_t s0, int64_t s1) { return ((uintptr_t)p & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0; }

/* tokens a warp takes at a time: as many as leave every warp of the GPU something to do */
uint32_t tokens_of_item(uint64_t n_tokens, uint32_t heads, uint64_t warps)
{
    uint32_t t = KV_MAX_LANE_TOKENS;
    while (t > 1 && (n_tokens + t - 1) / t * heads < warps) t >>= 1;
    return t;
}

}  // namespace

extern "C" uint64_t bam_kv_scratch_bytes(bam_array_t a, const bam_kv_layout_t* layout)
{
    kv_layout_d_t L;
    if (kv_layout(a, layout, &L) != BAM_OK) return 0;
    const uint32_t most = kv_most_blocks(a);
    return kv_parts_at(most * KV_WORKERS) + (uint64_t)most * KV_WORKERS * 2 * KV_ROWS * (L.head_dim + 2) * sizeof(float);
}

static int check_scratch(bam_array_t a, const bam_kv_layout_t* layout, void* scratch, uint64_t scratch_bytes)
{
    if (!scratch || ((uintptr_t)scratch & 127)) return BAM_EINVAL;
    return scratch_bytes < bam_kv_scratch_bytes(a, layout) ? BAM_EINVAL : BAM_OK;
}

template <class T>
static int launch_append(bam_array_t a, const kv_layout_d_t& L, const bam_kv_append_t* p, void* scratch, void* stream)
{
    KvAppendWork<T> w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.q = (const uint16_t*)p->q; w.k = (const uint16_t*)p->k; w.v = (const uint16_t*)p->v; w.q_out = (uint16_t*)p->q_out;
    w.q_st = p->q_stride[0]; w.q_sh = p->q_stride[1]; w.k_st = p->k_stride[0]; w.k_sh = p->k_stride[1];
    w.v_st = p->v_stride[0]; w.v_sh = p->v_stride[1]; w.qo_st = p->q_out_stride[0]; w.qo_sh = p->q_out_stride[1];
    w.n_tokens = p->n_tokens; w.n_q_heads = p->q ? p->n_q_heads : 0;
    w.lanes_per_row = lanes_of_row(L.chunks);
    const uint64_t warps = (uint64_t)a->pc->ctrl->num_sms * w.min_blocks * (w.threads / 32);
    w.tokens_per_item = tokens_of_item(p->n_tokens, L.n_kv_heads, warps);
    w.vec = (on_16(p->q, p->q_stride[0], p->q_stride[1]) ? 1u : 0u) | (on_16(p->k, p->k_stride[0], p->k_stride[1]) ? 2u : 0u) |
            (on_16(p->v, p->v_stride[0], p->v_stride[1]) ? 4u : 0u) | (on_16(p->q_out, p->q_out_stride[0], p->q_out_stride[1]) ? 8u : 0u);
    w.slots = p->slots;
    w.rope.positions = p->positions; w.rope.cos = p->cos; w.rope.sin = p->sin; w.rope.n_positions = p->n_positions;
    w.rope.stride = p->rope_stride; w.rope.rotary_dim = p->cos ? p->rotary_dim : 0; w.rope.style = p->rope_style;
    w.q_norm = (const uint16_t*)p->q_norm; w.k_norm = (const uint16_t*)p->k_norm; w.eps = p->norm_eps;
    const uint64_t items = (p->n_tokens + w.tokens_per_item - 1) / w.tokens_per_item * L.n_kv_heads;
    const uint64_t q_items = (p->n_tokens * w.n_q_heads + 32 / w.lanes_per_row - 1) / (32 / w.lanes_per_row);
    const uint64_t most = items > q_items ? items : q_items;
    return kv_launch(a->pc->ctrl, w, (most + w.threads / 32 - 1) / (w.threads / 32), scratch, sizeof(kv_launch_words_t), (cudaStream_t)stream);
}

extern "C" int bam_launch_kv_append(bam_array_t a, const bam_kv_layout_t* layout, const bam_kv_append_t* p, void* scratch_dev,
                                    uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!p || !p->k || !p->v || !p->slots || p->n_tokens > 0x7fffffffull) return BAM_EINVAL;
    if (p->q && (!p->q_out || p->n_q_heads == 0 || p->n_q_heads > 65536)) return BAM_EINVAL;
    if (p->cos || p->sin) {
        if (!p->cos || !p->sin || !p->positions || p->n_positions == 0 || p->n_positions > 0x7fffffffffffull) return BAM_EINVAL;
        if (p->rotary_dim == 0 || p->rotary_dim > L.head_dim || p->rotary_dim % 16 || p->rope_stride < p->rotary_dim / 2) return BAM_EINVAL;
        if (p->rope_style != BAM_KV_ROPE_HALF && p->rope_style != BAM_KV_ROPE_PAIRS) return BAM_EINVAL;
    }
    if ((p->q_norm || p->k_norm) && !(p->norm_eps >= 0.f)) return BAM_EINVAL;
    rc = check_scratch(a, layout, scratch_dev, scratch_bytes);
    if (rc) return rc;
    if (p->n_tokens == 0) return BAM_OK;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    return layout->dtype == BAM_KV_BF16 ? launch_append<__nv_bfloat16>(a, L, p, scratch_dev, stream)
                                        : launch_append<__half>(a, L, p, scratch_dev, stream);
}

extern "C" int bam_launch_kv_gather(bam_array_t a, const bam_kv_layout_t* layout, uint64_t n_tokens, const int64_t* slots_dev,
                                    void* k_out_dev, void* v_out_dev, const int64_t* k_stride, const int64_t* v_stride,
                                    void* scratch_dev, uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!slots_dev || !k_out_dev || !v_out_dev || !k_stride || !v_stride || n_tokens > 0x7fffffffull) return BAM_EINVAL;
    rc = check_scratch(a, layout, scratch_dev, scratch_bytes);
    if (rc) return rc;
    if (n_tokens == 0) return BAM_OK;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    KvGatherWork w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.k = (uint16_t*)k_out_dev; w.v = (uint16_t*)v_out_dev;
    w.k_st = k_stride[0]; w.k_sh = k_stride[1]; w.v_st = v_stride[0]; w.v_sh = v_stride[1];
    w.n_tokens = n_tokens;
    w.lanes_per_row = lanes_of_row(L.chunks);
    const uint64_t warps = (uint64_t)a->pc->ctrl->num_sms * w.min_blocks * (w.threads / 32);
    w.tokens_per_item = tokens_of_item(n_tokens, L.n_kv_heads, warps);
    w.vec = (on_16(k_out_dev, k_stride[0], k_stride[1]) ? 1u : 0u) | (on_16(v_out_dev, v_stride[0], v_stride[1]) ? 2u : 0u);
    w.slots = slots_dev;
    const uint64_t items = (n_tokens + w.tokens_per_item - 1) / w.tokens_per_item * L.n_kv_heads;
    return kv_launch(a->pc->ctrl, w, (items + w.threads / 32 - 1) / (w.threads / 32), scratch_dev, sizeof(kv_launch_words_t), (cudaStream_t)stream);
}

extern "C" int bam_launch_kv_attend(bam_array_t a, const bam_kv_layout_t* layout, const bam_kv_attend_t* p, void* scratch_dev,
                                    uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!p || !p->q || !p->out || !p->block_table || !p->seq_lens) return BAM_EINVAL;
    if (p->n_q_heads == 0 || p->n_q_heads > 65536 || p->n_q_heads % L.n_kv_heads) return BAM_EINVAL;
    if (p->batch > (1u << 20) || p->table_width == 0 || p->table_width > (1u << 27) || p->window < 0 || p->sinks < 0) return BAM_EINVAL;
    if (!(p->scale == p->scale)) return BAM_EINVAL;
    rc = check_scratch(a, layout, scratch_dev, scratch_bytes);
    if (rc) return rc;
    if (p->batch == 0) return BAM_OK;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    return layout->dtype == BAM_KV_BF16 ? kv_launch_attend<__nv_bfloat16>(a, L, p, scratch_dev, stream)
                                        : kv_launch_attend<__half>(a, L, p, scratch_dev, stream);
}
