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
        /* rows of one page share a pin (the coalescing of the array reads) */
        const uint32_t eq = __match_any_sync(full, pending ? page : ~(uint64_t)lane);
        const uint32_t leader = __ffs(eq) - 1, cnt = __popc(eq);
        uint32_t slot = L.r.acquire_page_warp(full, pending && lane == leader, pending ? page : 0, cnt, write, queue);
        slot = __shfl_sync(full, slot, leader);
        const bool got = pending && slot <= BAM_SLOT_MAX;
        const bool failed = __any_sync(full, pending && slot == BAM_SLOT_ERR);
        const uint32_t m = __ballot_sync(full, got);
        if (m && !failed) rows(m, got ? L.r.get_cache_page_addr(slot) : 0);
        if (write) __threadfence();
        __syncwarp();
        if (got && lane == leader) L.r.release_page(slot, cnt);
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
/* attention of one new token per sequence                                                 */
/* ====================================================================================== */

/* The flattened work list: sequence b has `n` chunks of CS tokens with something visible in them, in each of its
 * n_kv_heads * tiles units (a unit: 16 query heads of one key/value head), and the list is b-major, then unit, then
 * chunk.  Worker block i takes the chunks [i * per, (i + 1) * per): every block reads the same amount whatever the
 * lengths are, a long sequence is split over many blocks and a short one is not split at all.  A block that does not
 * own a whole unit writes its running maximum, denominator and unnormalised sum to the scratch; the blocks of a unit
 * wait for each other at the end (they are co-resident, one cooperative launch) and each joins a part of the output,
 * adding in a fixed order: the same bits on every run.
 *
 * What bounds it is reading keys and values once from HBM: 4 head_dim bytes a token for 4 head_dim flops a query head,
 * 8 flops a byte at 8 query heads.  So the design feeds bulk copies: a producer warp looks pages up and pins them 32
 * at a time and copies each chunk's rows, keys and values, into a ring of shared memory stages; four consumer warps
 * take the chunks in turn, unpin the page as soon as its rows have landed, and keep one running softmax each, merged
 * once per unit.  The products go through m16n8k16 matrix instructions: 16 query heads are all the rows there are, at
 * a rate of a few percent of the tensor pipe, so the 128-row tcgen05 tiles would be seven eighths padding. */
#define KV_STAGES_MAX 24u
#define KV_CONSUMERS 4u
#define KV_ROWS 16u                   /* query heads of a unit: the rows of a matrix instruction */
#define KV_MIN_CHUNKS 4u              /* a block takes at least so many: below that splitting costs more than it saves */

struct kv_seen_t {
    int64_t len, first, begin;        /* visible: j < first, and begin <= j < len */
    uint32_t n_first, from, n;        /* chunks [0, n_first) and then [from, from + n - n_first) of the sequence */
};

BAM_DEV void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
BAM_DEV void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
BAM_DEV void ldm_x4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
BAM_DEV void ldm_x4_t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
BAM_DEV void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
BAM_DEV bool mbar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
BAM_DEV void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
BAM_DEV void st_cg_f4(float* p, float x, float y, float z, float w)
{
    asm volatile("st.global.cg.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
BAM_DEV void st_cg_f2(float* p, float x, float y) { asm volatile("st.global.cg.v2.f32 [%0], {%1,%2};" ::"l"(p), "f"(x), "f"(y) : "memory"); }
BAM_DEV float ld_cg_f(const float* p) { float v; asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory"); return v; }

/* Shared memory of a worker block behind its ring of stages. */
template <int DMAX>
struct kv_shared_t {
    float merge[2][KV_ROWS][DMAX];            /* two warps' sums on their way into two others         */
    float m[KV_CONSUMERS][KV_ROWS], l[KV_CONSUMERS][KV_ROWS];
    uint64_t full[KV_STAGES_MAX], empty[KV_STAGES_MAX];
    uint32_t pin[KV_STAGES_MAX];              /* cache slot that is pinned for the stage's rows       */
    uint64_t warp_sum[8];
    uint64_t total, start_pos;
    uint32_t start_b, issued;
    volatile uint32_t abort;
    uint32_t n_join;
    struct { uint32_t b, u; uint64_t first; uint32_t n; } join[2];
};

/* DMAX: the head_dim the registers are laid out for; CS: tokens of a chunk (it divides block_tokens). */
template <class T, int DMAX, int CS>
struct KvAttendWork {
    static constexpr int threads = 32 * (KV_CONSUMERS + 1), min_blocks = 2;
    static constexpr uint32_t smem = 112 * 1024;
    static constexpr uint32_t ring_bytes = (smem - (uint32_t)sizeof(kv_shared_t<DMAX>)) & ~1023u;
    static constexpr bool q_in_regs = DMAX <= 128;       /* at 256 the sums alone take 128 registers: the query is re-read (L1) */
    kv_layout_d_t L;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    int64_t q_sb, q_sh, o_sb, o_sh, table_stride;
    const int32_t *table, *lens;
    uint32_t batch, n_q_heads, table_width;
    uint32_t q32, o32;                                   /* two elements at a time lie on 4-byte boundaries */
    uint32_t group, tiles;                               /* query heads of a key/value head, units they make */
    float scale_log2;
    int64_t window, sinks;
    uint32_t* arrived;                                   /* per worker block, all ones at the start: arrivals at the unit it begins */
    float* parts;                                        /* [worker block][2]: head_dim x 16 sums, 16 maxima, 16 denominators */

    BAM_DEV uint32_t stages() const
    {
        const uint32_t n = ring_bytes / (CS * L.head_dim * 4u);
        return n < KV_STAGES_MAX ? n : KV_STAGES_MAX;
    }
    BAM_DEV float* part(uint32_t block, uint32_t which) const { return parts + ((size_t)block * 2 + which) * (KV_ROWS * (L.head_dim + 2)); }

    BAM_DEV kv_seen_t seen(uint32_t b, bool tell = false) const
    {
        kv_seen_t v;
        v.len = __ldg(lens + b);
        if (v.len < 0 || v.len > (int64_t)table_width * L.block_tokens) {
            if (tell) L.bad_index((uint64_t)v.len);
            v.len = 0;
        }
        v.first = v.begin = v.len;
        if (window > 0 && window < v.len) {
            const int64_t w0 = v.len - window;
            v.first = sinks < v.len ? sinks : v.len;
            if (w0 > v.first) v.begin = w0; else v.first = v.begin = v.len;
        }
        v.n_first = (uint32_t)((v.first + CS - 1) / CS);
        v.from = (uint32_t)(v.begin / CS);
        if (v.from < v.n_first) v.from = v.n_first;
        const uint32_t end = (uint32_t)((v.len + CS - 1) / CS);
        v.n = v.n_first + (end > v.from ? end - v.from : 0u);
        return v;
    }
    BAM_DEV static int64_t first_token(const kv_seen_t& v, uint32_t c) { return (int64_t)(c < v.n_first ? c : v.from + (c - v.n_first)) * CS; }

    /* A wait that ends: false when the block gives up (someone's wait ran out, or the status block says so). */
    BAM_DEV bool wait(kv_shared_t<DMAX>& sh, uint32_t bar, uint32_t parity) const
    {
        uint32_t polls = 0;
        uint64_t t0 = 0;
        while (!mbar_try(bar, parity)) {
            if (sh.abort) return false;
            if (((++polls) & 63u) == 0u) {
                bam_status_t* st = L.r.cache.status;
                const uint64_t now = global_timer_ns();
                if (t0 == 0) t0 = now;
                /* the producer's own waits have one limit each; twice that is more than it needs to report */
                if (now - t0 > 2 * st->spin_timeout_ns) status_fail(st, BAM_ETIMEDOUT, BAM_AT_TMA, bar);
                if (status_bad(st)) { sh.abort = 1; return false; }
            }
        }
        return true;
    }

    /* ---- producer ------------------------------------------------------------------------------------ */
    BAM_DEV void produce(kv_shared_t<DMAX>& sh, uint32_t ring, uint64_t f0, uint64_t f1, uint32_t vb) const
    {
        const uint32_t full_mask = 0xffffffffu, lane = lane_id();
        const uint32_t S = stages(), stage_bytes = CS * L.head_dim * 4u, units = L.n_kv_heads * tiles;
        uint32_t base_b = sh.start_b;
        uint64_t base_pos = sh.start_pos;
        spin_t sp;
        for (uint64_t f = f0; f < f1; f += 32) {
            bool pending = f + lane < f1;
            /* where this lane's chunk is */
            uint32_t b = base_b, rows = 0, row0 = 0, row_at = 0;
            uint64_t pos = base_pos + lane, page = 0;
            bool bad = false;
            if (pending) {
                kv_seen_t v = seen(b);
                while (pos >= (uint64_t)v.n * units && b + 1 < batch) { pos -= (uint64_t)v.n * units; v = seen(++b); }
                if (v.n == 0) { sh.abort = 1; v.n = 1; }                   /* the lengths changed under the launch */
                const uint32_t u = (uint32_t)(pos / v.n), c = (uint32_t)(pos - (uint64_t)u * v.n);
                const int64_t t0 = first_token(v, c);
                int64_t lo = t0, hi = t0 + CS < v.len ? t0 + CS : v.len;
                if (t0 >= v.first && lo < v.begin) lo = v.begin;
                if (t0 + CS <= v.begin && hi > v.first) hi = v.first;
                const int64_t block = __ldg(table + b * table_stride + t0 / L.block_tokens);
                bad = block < 0 || (uint64_t)block >= L.n_blocks;
                if (bad) L.bad_index((uint64_t)block);
                else page = L.page_of((uint64_t)block, u / tiles);
                rows = (uint32_t)(hi - lo);
                row0 = (uint32_t)(lo - t0);
                row_at = (uint32_t)(lo % L.block_tokens);
            }
            base_b = __shfl_sync(full_mask, b, 31);
            base_pos = __shfl_sync(full_mask, pos, 31) + 1;
            /* pin: chunks of one page share a fetch-add; a lane whose page cannot be had now is asked for again when
             * the chunks before it are under way, and the chunks behind it give theirs back meanwhile */
            sp.reset();
            for (;;) {
                const uint32_t todo = __ballot_sync(full_mask, pending);
                if (todo == 0u) break;
                const bool want = pending && !bad;
                const uint32_t eq = __match_any_sync(full_mask, want ? page : ~(uint64_t)lane);
                const uint32_t leader = __ffs(eq) - 1;
                uint32_t slot = L.r.acquire_page_warp(full_mask, want && lane == leader, want ? page : 0, __popc(eq), false, vb * 8u);
                slot = __shfl_sync(full_mask, slot, leader);
                const bool got = want && slot <= BAM_SLOT_MAX;
                const uint32_t miss = __ballot_sync(full_mask, want && !got);
                const uint32_t last = miss ? __ffs(miss) - 1 : 32u;                /* lanes below go out now */
                const bool failed = __any_sync(full_mask, want && slot == BAM_SLOT_ERR);
                if (got && (lane >= last || failed)) L.r.release_page(slot, 1);
                if (failed) { sh.abort = 1; __syncwarp(); return; }
                /* what was filled in this launch came through the same kind of bulk copies; order them before ours */
                asm volatile("fence.proxy.async.global;" ::: "memory");
                const uint64_t src = got ? L.r.get_cache_page_addr(slot) + row_at * L.row_bytes() : 0;
                bool ok = true;
                for (uint32_t i = __ffs(todo) - 1; i < last && ((todo >> i) & 1u); i++) {
                    if (lane == i) {
                        const uint32_t k = (uint32_t)(f - f0) + i, s = k % S, use = k / S;
                        const uint32_t full = smem_u32(&sh.full[s]);
                        ok = wait(sh, smem_u32(&sh.empty[s]), (use & 1u) ^ 1u);
                        if (ok) {
                            sh.pin[s] = bad ? BAM_SLOT_NONE : slot;
                            if (bad) mbar_arrive(full);
                            else {
                                const uint32_t bytes = rows * L.row_bytes(), dst = ring + s * stage_bytes + row0 * L.row_bytes();
                                mbar_expect_tx(full, 2 * bytes);
                                bulk_load(dst, reinterpret_cast<const void*>(src), bytes, full);
                                bulk_load(dst + CS * L.row_bytes(), reinterpret_cast<const void*>(src + L.v_offset()), bytes, full);
                            }
                            sh.issued = k + 1;
                        } else if (got) L.r.release_page(slot, 1);
                        pending = false;
                    }
                    __syncwarp();
                }
                if (__any_sync(full_mask, !ok)) return;
                if (miss && last == (uint32_t)(__ffs(todo) - 1) && __any_sync(full_mask, sp.expired(L.r.cache.status, BAM_AT_FIND_SLOT, page))) {
                    sh.abort = 1;
                    __syncwarp();
                    return;
                }
            }
        }
    }

    /* ---- consumers ----------------------------------------------------------------------------------- */
    BAM_DEV uint32_t q_pair(const uint16_t* row, uint32_t d) const
    {
        if (q32) return __ldg(reinterpret_cast<const uint32_t*>(row + d));
        return (uint32_t)__ldg(row + d) | ((uint32_t)__ldg(row + d + 1) << 16);
    }
    /* the query fragment of dimensions [16 ks, 16 ks + 16): rows lane / 4 and lane / 4 + 8 */
    BAM_DEV void load_q(uint32_t (&a)[4], const uint16_t* r0, const uint16_t* r1, uint32_t ks) const
    {
        const uint32_t d = ks * 16 + (lane_id() & 3u) * 2;
        a[0] = r0 ? q_pair(r0, d) : 0u;
        a[1] = r1 ? q_pair(r1, d) : 0u;
        a[2] = r0 ? q_pair(r0, d + 8) : 0u;
        a[3] = r1 ? q_pair(r1, d + 8) : 0u;
    }

    struct state_t {
        float o[DMAX / 8][4];
        float m[2], l[2];
    };

    /* One chunk: S = Q K^T, p = 2^(S scale log2(e) - m), O += p V.  The weights go into the product as two 16-bit
     * parts, p = hi + lo, which keeps 16 (bf16) or more bits of them: the product runs twice, on a pipe that idles. */
    BAM_DEV void chunk(state_t& z, const uint32_t (&qa)[q_in_regs ? DMAX / 16 : 1][4], const uint16_t* q0, const uint16_t* q1, uint32_t stage,
                       const kv_seen_t& v, int64_t t0) const
    {
        const uint32_t lane = lane_id(), rb = L.row_bytes();
        const uint32_t x = ((lane & 7u) >> L.swz_shift) & L.swz_mask;
        const bool whole = t0 + CS <= v.first || (t0 >= v.begin && t0 + CS <= v.len);
        float s[CS / 8][4];
#pragma unroll
        for (int i = 0; i < CS / 8; i++) { s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f; }
        const uint32_t k_row = stage + ((lane & 7u) + ((lane >> 4) & 1u) * 8u) * rb, k_c = (lane >> 3) & 1u;
#pragma unroll
        for (int ks = 0; ks < DMAX / 16; ks++) {
            if (ks * 16 < (int)L.head_dim) {
                uint32_t a[4];
                if (q_in_regs) { a[0] = qa[q_in_regs ? ks : 0][0]; a[1] = qa[q_in_regs ? ks : 0][1]; a[2] = qa[q_in_regs ? ks : 0][2]; a[3] = qa[q_in_regs ? ks : 0][3]; }
                else load_q(a, q0, q1, ks);
#pragma unroll
                for (int np = 0; np < CS / 16; np++) {
                    uint32_t r[4];
                    ldm_x4(r, k_row + np * 16 * rb + ((ks * 2 + k_c) ^ x) * 16u);
                    mma_16816(s[2 * np], a, r[0], r[1], T());
                    mma_16816(s[2 * np + 1], a, r[2], r[3], T());
                }
            }
        }
        /* bit i: this lane's column i (of its CS / 4) is visible */
        uint32_t vis = 0xffffffffu;
        if (!whole) {
            vis = 0;
#pragma unroll
            for (int i = 0; i < CS / 4; i++) {
                const int64_t j = t0 + (i >> 1) * 8 + (lane & 3u) * 2 + (i & 1);
                if ((j < v.first || j >= v.begin) && j < v.len) vis |= 1u << i;
            }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < CS / 8; i++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[i][e] *= scale_log2;
                if (!((vis >> (2 * i + (e & 1))) & 1u)) s[i][e] = -INFINITY;
            }
            mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][1]));
            mx1 = fmaxf(mx1, fmaxf(s[i][2], s[i][3]));
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float n0 = fmaxf(z.m[0], mx0), n1 = fmaxf(z.m[1], mx1);
        const float c0 = n0 == -INFINITY ? 0.f : n0, c1 = n1 == -INFINITY ? 0.f : n1;     /* nothing seen yet: exp2(-inf - 0) = 0 */
        if (__any_sync(0xffffffffu, n0 != z.m[0] || n1 != z.m[1])) {
            const float a0 = exp2f(z.m[0] - c0), a1 = exp2f(z.m[1] - c1);
            z.l[0] *= a0; z.l[1] *= a1;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) { z.o[i][0] *= a0; z.o[i][1] *= a0; z.o[i][2] *= a1; z.o[i][3] *= a1; }
            z.m[0] = n0; z.m[1] = n1;
        }
        const uint32_t v_row = stage + CS * rb + ((lane & 7u) + ((lane >> 3) & 1u) * 8u) * rb, v_c = (lane >> 4) & 1u;
#pragma unroll
        for (int kt = 0; kt < CS / 16; kt++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; e++) p[e] = exp2f(s[2 * kt + half][e] - (e < 2 ? c0 : c1));
                z.l[0] += p[0] + p[1];
                z.l[1] += p[2] + p[3];
                hi[2 * half] = kv_type<T>::pack(p[0], p[1]);
                hi[2 * half + 1] = kv_type<T>::pack(p[2], p[3]);
                const float2 h0 = kv_type<T>::unpack(hi[2 * half]), h1 = kv_type<T>::unpack(hi[2 * half + 1]);
                lo[2 * half] = kv_type<T>::pack(p[0] - h0.x, p[1] - h0.y);
                lo[2 * half + 1] = kv_type<T>::pack(p[2] - h1.x, p[3] - h1.y);
            }
            /* rows that are not visible may hold anything, and 0 x NaN is not 0: they become zeros */
            uint32_t k0 = 0xffffffffu, k1 = 0xffffffffu;
            if (!whole) {
                const uint32_t bits = vis >> (4 * kt);
                k0 = ((bits & 1u) ? 0x0000ffffu : 0u) | ((bits & 2u) ? 0xffff0000u : 0u);
                k1 = ((bits & 4u) ? 0x0000ffffu : 0u) | ((bits & 8u) ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int np = 0; np < DMAX / 16; np++) {
                if (np * 16 < (int)L.head_dim) {
                    uint32_t r[4];
                    ldm_x4_t(r, v_row + kt * 16 * rb + ((np * 2 + v_c) ^ x) * 16u);
                    if (!whole) { r[0] &= k0; r[1] &= k1; r[2] &= k0; r[3] &= k1; }
                    mma_16816(z.o[2 * np], hi, r[0], r[1], T());
                    mma_16816(z.o[2 * np + 1], hi, r[2], r[3], T());
                    mma_16816(z.o[2 * np], lo, r[0], r[1], T());
                    mma_16816(z.o[2 * np + 1], lo, r[2], r[3], T());
                }
            }
        }
    }

    BAM_DEV void store_pair(uint16_t* p, float x, float y) const
    {
        const uint32_t w = kv_type<T>::pack(x, y);
        if (o32) *reinterpret_cast<uint32_t*>(p) = w;
        else { p[0] = (uint16_t)w; p[1] = (uint16_t)(w >> 16); }
    }
    BAM_DEV static float lse_of(float m, float l) { return m == -INFINITY ? -INFINITY : m * 0.69314718055994531f + logf(l); }

    /* the unit's result from one warp's registers */
    BAM_DEV void write_out(const state_t& z, uint32_t b, uint32_t u) const
    {
        const uint32_t lane = lane_id(), h = u / tiles, r0 = (u - h * tiles) * KV_ROWS;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = r0 + (lane >> 2) + 8 * half;
            if (r < group) {
                const uint32_t hq = h * group + r;
                const float inv = z.l[half] == 0.f ? 0.f : 1.f / z.l[half];
                uint16_t* p = out + b * o_sb + hq * o_sh + (lane & 3u) * 2;
#pragma unroll
                for (int i = 0; i < DMAX / 8; i++)
                    if (i * 8 < (int)L.head_dim) store_pair(p + i * 8, z.o[i][2 * half] * inv, z.o[i][2 * half + 1] * inv);
                if (lse && (lane & 3u) == 0u) lse[(size_t)b * n_q_heads + hq] = lse_of(z.m[half], z.l[half]);
            }
        }
    }
    BAM_DEV void write_part(const state_t& z, float* p) const
    {
        const uint32_t lane = lane_id();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = (lane >> 2) + 8 * half;
            float* row = p + r * L.head_dim + (lane & 3u) * 2;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++)
                if (i * 8 < (int)L.head_dim) st_cg_f2(row + i * 8, z.o[i][2 * half], z.o[i][2 * half + 1]);
            if ((lane & 3u) == 0u) {
                float* ml = p + KV_ROWS * L.head_dim;
                ml[r] = z.m[half];
                ml[KV_ROWS + r] = z.l[half];
            }
        }
    }

    /* Merge the consumers' states into warp 0's. */
    BAM_DEV void merge(kv_shared_t<DMAX>& sh, state_t& z, uint32_t w) const
    {
        const uint32_t lane = lane_id(), row = lane >> 2;
        if ((lane & 3u) == 0u) {
#pragma unroll
            for (int half = 0; half < 2; half++) { sh.m[w][row + 8 * half] = z.m[half]; sh.l[w][row + 8 * half] = z.l[half]; }
        }
        consumers_sync();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = row + 8 * half;
            float M = -INFINITY, l = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < KV_CONSUMERS; k++) M = fmaxf(M, sh.m[k][r]);
            const float c = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (uint32_t k = 0; k < KV_CONSUMERS; k++) l += sh.l[k][r] * exp2f(sh.m[k][r] - c);
            const float a = exp2f(z.m[half] - c);
            z.m[half] = M;
            z.l[half] = l;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) { z.o[i][2 * half] *= a; z.o[i][2 * half + 1] *= a; }
        }
        auto put = [&](uint32_t k) {
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) {
                if (i * 8 < (int)L.head_dim) {
                    float* p = &sh.merge[k][row][i * 8 + (lane & 3u) * 2];
                    *reinterpret_cast<float2*>(p) = make_float2(z.o[i][0], z.o[i][1]);
                    *reinterpret_cast<float2*>(p + 8 * DMAX) = make_float2(z.o[i][2], z.o[i][3]);
                }
            }
        };
        auto add = [&](uint32_t k) {
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) {
                if (i * 8 < (int)L.head_dim) {
                    const float* p = &sh.merge[k][row][i * 8 + (lane & 3u) * 2];
                    const float2 x = *reinterpret_cast<const float2*>(p), y = *reinterpret_cast<const float2*>(p + 8 * DMAX);
                    z.o[i][0] += x.x; z.o[i][1] += x.y; z.o[i][2] += y.x; z.o[i][3] += y.y;
                }
            }
        };
        if (w >= 2) put(w - 2);
        consumers_sync();
        if (w < 2) add(w);
        if (w == 1) put(1);
        consumers_sync();
        if (w == 0) add(1);
    }

    BAM_DEV void consume(kv_shared_t<DMAX>& sh, uint32_t ring, uint64_t f0, uint64_t f1, uint64_t per, uint32_t vb) const
    {
        const uint32_t lane = lane_id(), w = threadIdx.x >> 5;
        const uint32_t S = stages(), stage_bytes = CS * L.head_dim * 4u, units = L.n_kv_heads * tiles;
        uint32_t b = sh.start_b, n_join = 0;
        uint64_t pos = sh.start_pos;
        uint32_t stage = w % S, use = w / S;                  /* of this warp's next chunk: chunks w, w + 4, ... of the block */
        for (uint64_t f = f0; f < f1;) {
            const kv_seen_t v = seen(b);
            if (pos >= (uint64_t)v.n * units) {
                pos -= (uint64_t)v.n * units;
                if (++b >= batch) break;
                continue;
            }
            const uint32_t u = (uint32_t)(pos / v.n), c = (uint32_t)(pos - (uint64_t)u * v.n);
            const uint32_t seg = (uint32_t)(f1 - f < v.n - c ? f1 - f : v.n - c);
            const uint32_t h = u / tiles, r0 = (u - h * tiles) * KV_ROWS + (lane >> 2);
            const uint16_t* q0 = r0 < group ? q + b * q_sb + (int64_t)(h * group + r0) * q_sh : nullptr;
            const uint16_t* q1 = r0 + 8 < group ? q + b * q_sb + (int64_t)(h * group + r0 + 8) * q_sh : nullptr;
            state_t z;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) z.o[i][0] = z.o[i][1] = z.o[i][2] = z.o[i][3] = 0.f;
            z.m[0] = z.m[1] = -INFINITY;
            z.l[0] = z.l[1] = 0.f;
            uint32_t qa[q_in_regs ? DMAX / 16 : 1][4];
            const uint32_t mine = (w - (uint32_t)(f - f0)) & (KV_CONSUMERS - 1u);          /* first chunk of the segment that is this warp's */
            if (q_in_regs && mine < seg) {
#pragma unroll
                for (int ks = 0; ks < (q_in_regs ? DMAX / 16 : 1); ks++)
                    if (ks * 16 < (int)L.head_dim) load_q(qa[ks], q0, q1, ks);
            }
            for (uint32_t i = mine; i < seg; i += KV_CONSUMERS) {
                if (__all_sync(0xffffffffu, wait(sh, smem_u32(&sh.full[stage]), use & 1u))) {
                    const uint32_t slot = sh.pin[stage];
                    __syncwarp();
                    if (lane == 0 && slot != BAM_SLOT_NONE) { sh.pin[stage] = BAM_SLOT_NONE; L.r.release_page(slot, 1); }
                    if (slot != BAM_SLOT_NONE) chunk(z, qa, q0, q1, ring + stage * stage_bytes, v, first_token(v, c + i));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.empty[stage]));
                }
                stage += KV_CONSUMERS;
                while (stage >= S) { stage -= S; use++; }
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {
                z.l[half] += __shfl_xor_sync(0xffffffffu, z.l[half], 1);
                z.l[half] += __shfl_xor_sync(0xffffffffu, z.l[half], 2);
            }
            if (seg > 1) merge(sh, z, w);
            const bool holds = seg > 1 ? w == 0 : mine == 0;
            if (seg == v.n) {
                if (holds) write_out(z, b, u);
            } else {
                const uint64_t U0 = f - c;
                const uint32_t i0 = (uint32_t)(U0 / per);
                if (holds) {
                    write_part(z, part(vb, vb == i0 ? 1 : 0));
                    __threadfence();
                    __syncwarp();
                    if (lane == 0 && !sh.abort) (void)atom_add_acq_rel(arrived + i0, 1u);
                    if (lane == 0) { sh.join[n_join].b = b; sh.join[n_join].u = u; sh.join[n_join].first = U0; sh.join[n_join].n = v.n; }
                }
                n_join++;
            }
            f += seg;
            pos += seg;
        }
        consumers_sync();
        for (uint32_t k = 0; k < n_join; k++) join(sh, sh.join[k].b, sh.join[k].u, sh.join[k].first, sh.join[k].n, per, vb);
    }

    /* This block's share of a unit that several blocks worked on. */
    BAM_DEV void join(kv_shared_t<DMAX>& sh, uint32_t b, uint32_t u, uint64_t U0, uint32_t n, uint64_t per, uint32_t vb) const
    {
        const uint32_t lane = lane_id(), w = threadIdx.x >> 5, D = L.head_dim;
        const uint32_t i0 = (uint32_t)(U0 / per), cnt = (uint32_t)((U0 + n - 1) / per) - i0 + 1, j = vb - i0;
        if (threadIdx.x == 0) {
            spin_t sp;
            while (ld_acquire_gpu(arrived + i0) != cnt - 1u) {
                if (sh.abort) break;
                if (sp.expired(L.r.cache.status, BAM_AT_KV_JOIN, i0)) { sh.abort = 1; break; }
            }
        }
        consumers_sync();
        if (__any_sync(0xffffffffu, sh.abort)) return;
        const uint32_t h = u / tiles, r0 = (u - h * tiles) * KV_ROWS;
        const uint32_t rows = group - r0 < KV_ROWS ? group - r0 : KV_ROWS, quads = rows * (D / 4);
        const uint32_t g0 = (uint32_t)((uint64_t)quads * j / cnt), g1 = (uint32_t)((uint64_t)quads * (j + 1) / cnt);
        uint32_t P = 1;
        while (P < cnt && P < 32u) P <<= 1;
        const uint32_t p = lane & (P - 1u), at_once = 32u / P * KV_CONSUMERS;
        for (uint32_t base = g0; base < g1; base += at_once) {
            const uint32_t gi = base + w * (32u / P) + lane / P;
            const bool act = gi < g1;
            const uint32_t r = act ? gi / (D / 4) : 0, d = act ? (gi - r * (D / 4)) * 4 : 0;
            float M = -INFINITY;
            for (uint32_t s = p; s < cnt; s += P) M = fmaxf(M, ld_cg_f(part(i0 + s, s == 0 ? 1 : 0) + KV_ROWS * D + r));
            for (uint32_t o = P >> 1; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            const float c = M == -INFINITY ? 0.f : M;
            float l = 0.f, x[4] = { 0.f, 0.f, 0.f, 0.f };
            for (uint32_t s = p; s < cnt; s += P) {
                const float* q_ = part(i0 + s, s == 0 ? 1 : 0);
                const float a = exp2f(ld_cg_f(q_ + KV_ROWS * D + r) - c);
                l += a * ld_cg_f(q_ + KV_ROWS * (D + 1) + r);
                const uint4 y = ld_cg_v4(q_ + r * D + d);
                x[0] += a * __uint_as_float(y.x); x[1] += a * __uint_as_float(y.y); x[2] += a * __uint_as_float(y.z); x[3] += a * __uint_as_float(y.w);
            }
            for (uint32_t o = P >> 1; o > 0; o >>= 1) {
                l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
            }
            if (act && p == 0) {
                const uint32_t hq = h * group + r0 + r;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t* dst = out + b * o_sb + hq * o_sh + d;
                store_pair(dst, x[0] * inv, x[1] * inv);
                store_pair(dst + 2, x[2] * inv, x[3] * inv);
                if (lse && d == 0) lse[(size_t)b * n_q_heads + hq] = lse_of(M, l);
            }
        }
    }

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        kv_shared_t<DMAX>& sh = *reinterpret_cast<kv_shared_t<DMAX>*>(bam_dyn_smem + ring_bytes);
        const uint32_t ring = smem_u32(bam_dyn_smem), t = threadIdx.x, lane = t & 31u, w = t >> 5;
        const uint32_t units = L.n_kv_heads * tiles, S = stages();
        if (t < S) {
            mbar_init(smem_u32(&sh.full[t]), 1);
            mbar_init(smem_u32(&sh.empty[t]), 1);
            sh.pin[t] = BAM_SLOT_NONE;
        }
        if (t == 0) { sh.abort = status_bad(L.r.cache.status) ? 1u : 0u; sh.issued = 0; }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        /* how many chunks there are before each sequence: every thread counts a run of sequences */
        const uint32_t run = (batch + threads - 1) / threads;
        const uint32_t s0 = t * run < batch ? t * run : batch, s1 = s0 + run < batch ? s0 + run : batch;
        uint64_t own = 0;
        for (uint32_t b = s0; b < s1; b++) own += seen(b, vb == 0).n;
        uint64_t before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= (uint32_t)o) before += x;
        }
        if (lane == 31) sh.warp_sum[w] = before;
        before -= own;
        __syncthreads();
        if (sh.abort) return;
        uint64_t total = 0;
#pragma unroll
        for (uint32_t k = 0; k < KV_CONSUMERS + 1; k++) {
            if (k < w) before += sh.warp_sum[k];
            total += sh.warp_sum[k];
        }
        total *= units;
        uint64_t per = (total + nvb - 1) / nvb;
        if (per < KV_MIN_CHUNKS) per = KV_MIN_CHUNKS;
        const uint64_t f0 = (uint64_t)vb * per, f1 = f0 + per < total ? f0 + per : total;
        if (own && f0 >= before * units && f0 < (before + own) * units) {
            uint64_t at = before * units;
            for (uint32_t b = s0; b < s1; b++) {
                const uint64_t span = (uint64_t)seen(b).n * units;
                if (f0 < at + span) { sh.start_b = b; sh.start_pos = f0 - at; break; }
                at += span;
            }
        }
        /* sequences with nothing visible */
        for (uint32_t b = vb; b < batch; b += nvb) {
            if (seen(b).n == 0) {
                for (uint32_t i = t; i < n_q_heads * L.chunks * 4; i += threads) {
                    const uint32_t hq = i / (L.chunks * 4);
                    store_pair(out + b * o_sb + hq * o_sh + (i - hq * (L.chunks * 4)) * 2, 0.f, 0.f);
                }
                if (lse) for (uint32_t i = t; i < n_q_heads; i += threads) lse[(size_t)b * n_q_heads + i] = -INFINITY;
            }
        }
        __syncthreads();
        if (f0 < f1) {
            if (w == KV_CONSUMERS) produce(sh, ring, f0, f1, vb);
            else consume(sh, ring, f0, f1, per, vb);
        }
        __syncthreads();
        if (sh.abort && t < S && sh.pin[t] != BAM_SLOT_NONE) {
            /* given up: a copy that is still under way lands (bounded) before the block leaves, then its page is unpinned */
            const uint32_t use = (sh.issued - 1u - t) / S;
            const uint64_t since = global_timer_ns();
            while (!mbar_test(smem_u32(&sh.full[t]), use & 1u) && global_timer_ns() - since < 2 * L.r.cache.status->spin_timeout_ns) {}
            L.r.release_page(sh.pin[t], 1);
        }
    }
};

/* ====================================================================================== */
/* host side                                                                               */
/* ====================================================================================== */

namespace {

/* The calling thread's device is the caller's affair: it is put back when the entry point returns. */
struct device_guard {
    int was = -1;
    cudaError_t enter(int dev)
    {
        cudaError_t e = cudaGetDevice(&was);
        if (e == cudaSuccess && was != dev) e = cudaSetDevice(dev);
        return e;
    }
    ~device_guard()
    {
        int now = -1;
        if (was >= 0 && cudaGetDevice(&now) == cudaSuccess && now != was) (void)cudaSetDevice(was);
    }
};

/* Blocks of a kernel that are co-resident on the current device, and the shared memory attribute: asked once. */
template <class Work>
cudaError_t kv_max_grid(int dev, uint32_t* grid)
{
    static uint32_t known[64] = {};                  /* the same value whoever writes it */
    if (dev < 64 && known[dev]) { *grid = known[dev]; return cudaSuccess; }
    int sms = 0, nb = 0;
    cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(bam_kv_fused<Work>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Work::smem);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&nb, bam_kv_fused<Work>, Work::threads, Work::smem);
    if (e != cudaSuccess) return e;
    *grid = (uint32_t)nb * (uint32_t)sms;
    if (dev < 64) known[dev] = *grid;
    return cudaSuccess;
}

/* Launch with at most `want` worker blocks.  The launch's words are the first bytes of `scratch`; `clear` bytes of
 * it are set to all ones. */
template <class Work>
int kv_launch(bam_ctrl* c, const Work& work, uint64_t want, void* scratch, size_t clear, cudaStream_t s)
{
    uint32_t grid = 0;
    CK(kv_max_grid<Work>(c->device, &grid));
    if (c->max_grid && grid > c->max_grid) grid = c->max_grid;
    bam_emu_d_t emu = c->emu;
    if (want == 0) want = 1;
    /* few workers need few command processors, and a small grid starts and ends sooner */
    if (emu.n_ctrl_blocks > 4 && emu.n_ctrl_blocks > want) emu.n_ctrl_blocks = want > 4 ? (uint32_t)want : 4u;
    if (grid <= emu.n_ctrl_blocks) return BAM_EINVAL;
    if (grid - emu.n_ctrl_blocks > want) grid = emu.n_ctrl_blocks + (uint32_t)want;
    emu.consumers_remaining = reinterpret_cast<uint32_t*>(scratch);
    Work w = work;
    w.L.words = reinterpret_cast<kv_launch_words_t*>(scratch);
    CK(cudaMemsetAsync(scratch, 0xff, clear, s));
    void* args[] = { (void*)&emu, (void*)&w };
    CK(cudaLaunchCooperativeKernel((const void*)bam_kv_fused<Work>, dim3(grid), dim3(Work::threads), args, Work::smem, s));
    return BAM_OK;
}

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

/* Scratch: the launch's words, a counter per worker block, the blocks' parts. */
uint32_t kv_most_blocks(bam_array* a) { return (uint32_t)a->pc->ctrl->num_sms * 2u; }
size_t kv_parts_at(uint32_t blocks) { return (sizeof(kv_launch_words_t) + 4 * (size_t)blocks + 127) / 128 * 128; }

}  // namespace

extern "C" uint64_t bam_kv_scratch_bytes(bam_array_t a, const bam_kv_layout_t* layout)
{
    kv_layout_d_t L;
    if (kv_layout(a, layout, &L) != BAM_OK) return 0;
    const uint32_t most = kv_most_blocks(a);
    return kv_parts_at(most) + (uint64_t)most * 2 * KV_ROWS * (L.head_dim + 2) * sizeof(float);
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

template <class T, int DMAX, int CS>
static int launch_attend_as(bam_array_t a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    typedef KvAttendWork<T, DMAX, CS> Work;
    Work w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.q = (const uint16_t*)p->q; w.out = (uint16_t*)p->out; w.lse = p->lse;
    w.q_sb = p->q_stride[0]; w.q_sh = p->q_stride[1]; w.o_sb = p->out_stride[0]; w.o_sh = p->out_stride[1];
    w.table = p->block_table; w.table_stride = p->table_stride; w.table_width = p->table_width; w.lens = p->seq_lens;
    w.batch = p->batch; w.n_q_heads = p->n_q_heads;
    w.group = p->n_q_heads / L.n_kv_heads; w.tiles = (w.group + KV_ROWS - 1) / KV_ROWS;
    w.scale_log2 = p->scale * 1.4426950408889634f;
    w.window = p->window; w.sinks = p->sinks;
    w.q32 = ((uintptr_t)p->q & 3) == 0 && p->q_stride[0] % 2 == 0 && p->q_stride[1] % 2 == 0;
    w.o32 = ((uintptr_t)p->out & 3) == 0 && p->out_stride[0] % 2 == 0 && p->out_stride[1] % 2 == 0;
    uint8_t* base = (uint8_t*)scratch;
    const uint32_t most = kv_most_blocks(a);
    w.arrived = (uint32_t*)(base + sizeof(kv_launch_words_t));
    w.parts = (float*)(base + kv_parts_at(most));
    /* no more blocks than the longest sequences could keep busy */
    uint64_t chunks = (uint64_t)p->table_width * (L.block_tokens / CS);
    if (p->window > 0) {
        const uint64_t seen = (uint64_t)p->window / CS + (uint64_t)(p->sinks < (1ll << 40) ? p->sinks : (1ll << 40)) / CS + 4;
        if (seen < chunks) chunks = seen;
    }
    const uint64_t want = (chunks * p->batch * L.n_kv_heads * w.tiles + KV_MIN_CHUNKS - 1) / KV_MIN_CHUNKS;
    return kv_launch(a->pc->ctrl, w, want < most ? want : most, scratch, sizeof(kv_launch_words_t) + 4 * (size_t)most, (cudaStream_t)stream);
}

template <class T>
static int launch_attend(bam_array_t a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    const bool by32 = L.block_tokens % 32 == 0;
    if (L.head_dim <= 64) return by32 ? launch_attend_as<T, 64, 32>(a, L, p, scratch, stream) : launch_attend_as<T, 64, 16>(a, L, p, scratch, stream);
    if (L.head_dim <= 128) return by32 ? launch_attend_as<T, 128, 32>(a, L, p, scratch, stream) : launch_attend_as<T, 128, 16>(a, L, p, scratch, stream);
    return launch_attend_as<T, 256, 16>(a, L, p, scratch, stream);
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
    return layout->dtype == BAM_KV_BF16 ? launch_attend<__nv_bfloat16>(a, L, p, scratch_dev, stream)
                                        : launch_attend<__half>(a, L, p, scratch_dev, stream);
}
