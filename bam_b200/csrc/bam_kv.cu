/*
 * bam_kv.cu -- a key/value cache kept in the pages of an array: append (norm of each head and position rotation on
 * the way), gather, and attention of one new token per sequence.
 *
 * The reference has no counterpart: its consumers are graph and array kernels.  The pages are reached the way those
 * reach theirs -- look up, pin, read or write, unpin; a page that is not in the cache is fetched from the store
 * through the NVMe queues by the same launch -- so the rows of a cache larger than HBM need no other handling.
 */
#include <cuda_runtime.h>

#include <cmath>
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

/* A lane holds two 16-byte chunks of a row: the two halves of eight rotated pairs where there are such (chunks j and
 * j + rotary_dim / 16, or 2 j and 2 j + 1 for neighbouring pairs), so that a rotation needs no other lane and one set of
 * eight cosines and sines serves sixteen elements; they are loaded once per token and serve all its heads. */
struct kv_lane_t {
    uint32_t ca, cb;             /* the lane's chunks; ca = 0xffffffff: none                    */
    bool turned;                 /* they hold rotated pairs                                     */
    float c[8], s[8];            /* of the token at hand                                        */
    float w[16];                 /* the norm's weights, of the item at hand                     */
};

BAM_DEV kv_lane_t kv_lane(uint32_t j, uint32_t chunks, const kv_rope_d_t& rope)
{
    kv_lane_t n;
    const uint32_t half = rope.rotary_dim / 16;                        /* chunks of half the rotated elements */
    n.turned = j < half;
    if (n.turned && rope.style == BAM_KV_ROPE_HALF) { n.ca = j; n.cb = j + half; }
    else { n.ca = 2 * j; n.cb = 2 * j + 1; }                           /* rotary_dim and head_dim are multiples of 16 */
    if (n.cb >= chunks) n.ca = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 8; i++) { n.c[i] = 1.f; n.s[i] = 0.f; n.w[i] = n.w[8 + i] = 1.f; }
    return n;
}
template <bool VEC>
BAM_DEV void kv_load_angle(kv_lane_t& n, uint32_t j, const kv_rope_d_t& rope, int64_t pos)
{
    if (!n.turned || n.ca == 0xffffffffu) return;
    const float* c = rope.cos + pos * rope.stride + j * 8;
    const float* s = rope.sin + pos * rope.stride + j * 8;
    if (VEC) {
        const float4 c0 = __ldg(reinterpret_cast<const float4*>(c)), c1 = __ldg(reinterpret_cast<const float4*>(c) + 1);
        const float4 s0 = __ldg(reinterpret_cast<const float4*>(s)), s1 = __ldg(reinterpret_cast<const float4*>(s) + 1);
        n.c[0] = c0.x; n.c[1] = c0.y; n.c[2] = c0.z; n.c[3] = c0.w; n.c[4] = c1.x; n.c[5] = c1.y; n.c[6] = c1.z; n.c[7] = c1.w;
        n.s[0] = s0.x; n.s[1] = s0.y; n.s[2] = s0.z; n.s[3] = s0.w; n.s[4] = s1.x; n.s[5] = s1.y; n.s[6] = s1.z; n.s[7] = s1.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) { n.c[i] = __ldg(c + i); n.s[i] = __ldg(s + i); }
    }
}

/* y = x * rsqrt(mean(x^2) + eps) * w of the row that G lanes hold, then the rotation: in 32 bits, rounded once.  All
 * lanes of the warp call it. */
template <class T>
BAM_DEV void kv_transform(uint4& a, uint4& b, const kv_lane_t& n, uint32_t G, float inv_dim, bool norm, float eps,
                          const kv_rope_d_t& rope)
{
    if (!norm && rope.rotary_dim == 0) return;
    float x[8], y[8];
    {
        const uint32_t u[4] = { a.x, a.y, a.z, a.w }, v[4] = { b.x, b.y, b.z, b.w };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = kv_type<T>::unpack(u[i]), g = kv_type<T>::unpack(v[i]);
            x[2 * i] = f.x; x[2 * i + 1] = f.y; y[2 * i] = g.x; y[2 * i + 1] = g.y;
        }
    }
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i] + y[i] * y[i];
        for (uint32_t o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss * inv_dim + eps);
#pragma unroll
        for (int i = 0; i < 8; i++) { x[i] = x[i] * inv * n.w[i]; y[i] = y[i] * inv * n.w[8 + i]; }
    }
    if (n.turned) {
        if (rope.style == BAM_KV_ROPE_HALF) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float p = x[i], q = y[i];
                x[i] = p * n.c[i] - q * n.s[i];
                y[i] = q * n.c[i] + p * n.s[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = p * n.c[i] - q * n.s[i];
                x[2 * i + 1] = q * n.c[i] + p * n.s[i];
                p = y[2 * i]; q = y[2 * i + 1];
                y[2 * i] = p * n.c[4 + i] - q * n.s[4 + i];
                y[2 * i + 1] = q * n.c[4 + i] + p * n.s[4 + i];
            }
        }
    }
    a = make_uint4(kv_type<T>::pack(x[0], x[1]), kv_type<T>::pack(x[2], x[3]), kv_type<T>::pack(x[4], x[5]), kv_type<T>::pack(x[6], x[7]));
    b = make_uint4(kv_type<T>::pack(y[0], y[1]), kv_type<T>::pack(y[2], y[3]), kv_type<T>::pack(y[4], y[5]), kv_type<T>::pack(y[6], y[7]));
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
        __syncwarp();
        /* one release per page: the lowest of the lanes that share it gives all their counts back (what the other lanes wrote
         * comes before it by the barrier) */
        const uint32_t same = __match_any_sync(full, got ? slot : ~lane);
        if (got && lane == (uint32_t)(__ffs(same) - 1)) {
            /* rows that were read are in registers, or stored from there: there is nothing a release would have to wait for */
            if (write) L.r.release_page(slot, __popc(same));
            else red_add_relaxed(&L.r.cache.slots[slot].state, 0u - (uint32_t)__popc(same));
        }
        if (failed) return false;
        if (got) pending = false;
        if (m == 0u && __any_sync(full, sp.expired(L.r.cache.status, BAM_AT_FIND_SLOT, page))) return false;
    }
    return true;
}

/* The work is cut into items that warps draw in turn: first k_heads of the key/value heads of the runs that begin in k_tokens
 * consecutive tokens, then q_heads of the query heads of q_tokens tokens.  A run is the tokens in a row that go to one
 * block: one warp writes its share of it, to the end of the run and not of the item, and pins each page once.  (Warps that
 * miss the same page at once claim a slot each: a prompt whose pages were written by two warps each evicted half of a cache
 * with room for all.  The price is paid by large blocks, resident or not: with 1024 tokens a block, 16000 tokens of 8 heads
 * are work for 128 warps.)  Items differ in length, hence the drawing; which warp writes a row changes nothing in it.
 * Items are as large as still makes enough of them: a warp pins its pages together and loads angles and weights once an
 * item.  16000 tokens of 32 + 8 heads of 128, gathered again: 144 us with items of 32 and 4 heads, 152 with 16 and 1, 170 with
 * 8 query heads (which are too few rows in flight); 777 tokens of 15 + 3 heads of 256: 33 us with 1 key/value head, 37 with
 * 2, 41 with 4.
 * Bytes bound it, every row is read and written once; what that needs is rows in flight: four rows of a lane are loaded before
 * the first is worked on (two: 164 us instead of 150).  It reaches 3.5 TB/s, 0.53 of a copy (111 us for 393 MB without the
 * gather): 16 warps an SM, all that 128 registers allow, wait for their loads in turn and issue in 40 % of the cycles;
 * a second row of keys in flight spilled far more than the 28 bytes a thread that the kernel spills as it is (190 us), rows
 * prefetched through shared memory, 96 KB a block, took 156 us instead of 142.  200 tokens take 18 us in a graph, one token 13:
 * the start and the end of a cooperative launch and the look-ups. */
#define KV_ROWS_AHEAD 4

/* VEC: every row, weight and angle lies on a 16-byte boundary. */
template <class T, bool VEC>
struct KvAppendWork {
    static constexpr int threads = BAM_THREADS, min_blocks = 2;
    static constexpr uint32_t smem = BAM_FUSED_SMEM;
    kv_layout_d_t L;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh;      /* element strides of token and head */
    uint64_t n_tokens;
    uint32_t n_q_heads, lanes_per_row, k_tokens, q_tokens, k_heads, q_heads, k_parts, q_parts;
    const int64_t* slots;
    kv_rope_d_t rope;
    const uint16_t *q_norm, *k_norm;
    float eps, inv_dim;

    BAM_DEV uint32_t counters(uint32_t) const { return 0; }

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

    /* the block a token goes to; ~0: none, it is padding or its slot is no slot */
    BAM_DEV uint64_t block_of(uint64_t t) const
    {
        const int64_t slot = slots[t];
        if (slot < 0) return ~0ull;
        if ((uint64_t)slot >= L.n_blocks * L.block_tokens) { L.bad_index((uint64_t)slot); return ~0ull; }
        return (uint64_t)slot / L.block_tokens;
    }

    /* rows [0, n) of one token, head by head: heads h0 + r */
    BAM_DEV void queries(uint64_t t, uint32_t h0, uint32_t n, const kv_lane_t& ln, uint32_t G, uint32_t grp) const
    {
        const uint32_t rows = 32u / G;
        const uint16_t* src = q + (int64_t)t * q_st;
        uint16_t* dst = q_out + (int64_t)t * qo_st;
        for (uint32_t r0 = 0; r0 < n; r0 += rows * KV_ROWS_AHEAD) {
            uint4 a[KV_ROWS_AHEAD], b[KV_ROWS_AHEAD];
#pragma unroll
            for (int i = 0; i < KV_ROWS_AHEAD; i++) {
                const uint32_t r = r0 + i * rows + grp;
                a[i] = b[i] = make_uint4(0, 0, 0, 0);
                if (r < n && ln.ca != 0xffffffffu) {
                    a[i] = kv_load8(src + (h0 + r) * q_sh + ln.ca * 8, VEC);
                    b[i] = kv_load8(src + (h0 + r) * q_sh + ln.cb * 8, VEC);
                }
            }
#pragma unroll
            for (int i = 0; i < KV_ROWS_AHEAD; i++) {
                if (r0 + i * rows >= n) break;
                const uint32_t r = r0 + i * rows + grp;
                kv_transform<T>(a[i], b[i], ln, G, inv_dim, q_norm != nullptr, eps, rope);
                if (r < n && ln.ca != 0xffffffffu) {
                    kv_store8(dst + (h0 + r) * qo_sh + ln.ca * 8, a[i], VEC);
                    kv_store8(dst + (h0 + r) * qo_sh + ln.cb * 8, b[i], VEC);
                }
            }
        }
    }

    /* Keys and values of the tokens t1 + i, i in `run` (a mask of the first n_run), heads h0 .. h0 + nh of them whose pages
     * are there (lane h of mask m holds the page of head h0 + h; lane i the row and the position of token i). */
    BAM_DEV void keys(uint64_t t1, uint32_t run, uint32_t n_run, uint32_t h0, uint32_t nh, uint32_t m, uint64_t addr, uint32_t row, int64_t pos,
                      const kv_lane_t& item, uint32_t j, uint32_t G, uint32_t grp) const
    {
        const uint32_t full = 0xffffffffu, rows = 32u / G, n = n_run * nh;
        /* row r: token r / nh, head r % nh */
        auto place = [&](uint32_t r, uint32_t& i, uint32_t& h, uint8_t*& base, uint32_t& rr) {
            i = r / nh;
            h = r - i * nh;
            base = reinterpret_cast<uint8_t*>(__shfl_sync(full, addr, h & 31u));
            rr = __shfl_sync(full, row, i & 31u);
            return r < n && ((run >> (i & 31u)) & 1u) && ((m >> (h & 31u)) & 1u) && item.ca != 0xffffffffu;
        };
        kv_lane_t ln = item;
        for (uint32_t r0 = 0; r0 < n; r0 += rows) {                                  /* every row has its token's angles */
            uint32_t i, h, rr;
            uint8_t* dst;
            if (!place(r0 + grp, i, h, dst, rr)) dst = nullptr;
            const int64_t at = __shfl_sync(full, pos, i & 31u);
            uint4 a = make_uint4(0, 0, 0, 0), b = a, va = a, vb = a;
            if (dst) {
                const uint16_t* src = k + (int64_t)(t1 + i) * k_st + (h0 + h) * k_sh;
                a = kv_load8(src + item.ca * 8, VEC);
                b = kv_load8(src + item.cb * 8, VEC);
                kv_load_angle<VEC>(ln, j, rope, at);
                src = v + (int64_t)(t1 + i) * v_st + (h0 + h) * v_sh;
                va = kv_load8(src + item.ca * 8, VEC);
                vb = kv_load8(src + item.cb * 8, VEC);
            }
            kv_transform<T>(a, b, ln, G, inv_dim, k_norm != nullptr, eps, rope);
            if (dst) {
                uint8_t* p = dst + rr * L.row_bytes() + L.swizzle(rr, item.ca) * 16u;
                *reinterpret_cast<uint4*>(p) = a;
                *reinterpret_cast<uint4*>(p + L.v_offset()) = va;
                p = dst + rr * L.row_bytes() + L.swizzle(rr, item.cb) * 16u;
                *reinterpret_cast<uint4*>(p) = b;
                *reinterpret_cast<uint4*>(p + L.v_offset()) = vb;
            }
        }
    }

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        const uint32_t full = 0xffffffffu, lane = threadIdx.x & 31u;
        const uint64_t warp = (uint64_t)(threadIdx.x >> 5) * nvb + vb, nwarps = (uint64_t)nvb * (blockDim.x >> 5);
        const uint32_t G = lanes_per_row, j = lane & (G - 1u), grp = lane / G;
        if (status_bad(L.r.cache.status)) return;
        kv_lane_t ln = kv_lane(j, L.chunks, rope);
        const uint64_t k_items = (n_tokens + k_tokens - 1) / k_tokens * k_parts;
        const uint64_t n_items = k_items + (q_parts ? (n_tokens + q_tokens - 1) / q_tokens * q_parts : 0u);
        for (uint64_t it = warp; it < n_items; it = nwarps + L.draw()) {
            const bool queries_of = it >= k_items;
            const uint64_t x = queries_of ? it - k_items : it;
            const uint32_t parts = queries_of ? q_parts : k_parts, span = queries_of ? q_tokens : k_tokens;
            const uint32_t part = (uint32_t)(x % parts);
            const uint64_t t0 = x / parts * span;
            const uint32_t nt = n_tokens - t0 < span ? (uint32_t)(n_tokens - t0) : span;
            const uint16_t* norm = queries_of ? q_norm : k_norm;
            if (norm && ln.ca != 0xffffffffu) {
                const uint4 wa = kv_load8(norm + ln.ca * 8, VEC), wb = kv_load8(norm + ln.cb * 8, VEC);
                const uint32_t w[8] = { wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w };
#pragma unroll
                for (int i = 0; i < 8; i++) { const float2 f = kv_type<T>::unpack(w[i]); ln.w[2 * i] = f.x; ln.w[2 * i + 1] = f.y; }
            }
            if (queries_of) {
                const uint32_t h0 = part * q_heads, n = n_q_heads - h0 < q_heads ? n_q_heads - h0 : q_heads;
                const int64_t pos = lane < nt ? position(t0 + lane, slots[t0 + lane] < 0) : 0;
                for (uint32_t i = 0; i < nt; i++) {
                    const int64_t p = __shfl_sync(full, pos, i);
                    if (p < 0) continue;
                    kv_load_angle<VEC>(ln, j, rope, p);
                    queries(t0 + i, h0, n, ln, G, grp);
                }
                continue;
            }
            const uint64_t mine = lane < nt ? block_of(t0 + lane) : ~0ull;
            const uint64_t before = lane < nt && t0 + lane > 0 ? block_of(t0 + lane - 1) : ~0ull;
            for (uint32_t begins = __ballot_sync(full, mine != ~0ull && mine != before); begins; begins &= begins - 1) {
                const uint32_t first = __ffs(begins) - 1;
                const uint64_t at = __shfl_sync(full, mine, first);
                for (uint64_t t1 = t0 + first;; t1 += 32) {          /* 32 tokens of the run at a time */
                    const uint64_t t = t1 + lane;
                    const bool here = t < n_tokens && block_of(t) == at;
                    const uint32_t gap = ~__ballot_sync(full, here);
                    const uint32_t in_run = gap ? (1u << (__ffs(gap) - 1)) - 1u : full;
                    const bool live = (in_run >> lane) & 1u;
                    const int64_t pos = live ? position(t, false) : 0;
                    const uint32_t row = live ? (uint32_t)((uint64_t)slots[t] % L.block_tokens) : 0;
                    const uint32_t run = in_run & __ballot_sync(full, pos >= 0);
                    const uint32_t h0 = part * k_heads, nh = L.n_kv_heads - h0 < k_heads ? L.n_kv_heads - h0 : k_heads;
                    if (run && !kv_with_pages(L, lane < nh, L.page_of(at, h0 + lane), true, (uint32_t)warp, [&](uint32_t m, uint64_t addr) {
                            keys(t1, run, 32u - __clz(run), h0, nh, m, addr, row, pos, ln, j, G, grp);
                        })) return;
                    if (gap) break;
                }
            }
        }
    }
};

/* ====================================================================================== */
/* gather                                                                                  */
/* ====================================================================================== */

/* Items of up to 32 tokens of one head, drawn in turn: a lane looks up the page of a token, then groups of lanes copy rows.
 * Bytes bound it.  30001 tokens of 8 heads of 128 take 54 us, 4.6 TB/s: about 12 us of a launch that starts, looks its first
 * pages up and ends, and the rest at what a copy reaches.  Three blocks an SM, four rows of a lane loaded before the first
 * is stored (two: 65 us; eight at two blocks: 71).  Through shared memory with bulk copies, the look-ups of an item wait for
 * its one stage: 64 to 73 us.  80 registers, for three blocks an SM, spill 52 bytes a thread.  An indexing kernel over plain
 * tensors needs no look-up and takes 53 us; the rows of 200 tokens take 17 us in a graph. */
template <bool VEC>
struct KvGatherWork {
    static constexpr int threads = BAM_THREADS, min_blocks = 3;
    static constexpr uint32_t smem = BAM_FUSED_SMEM;
    kv_layout_d_t L;
    uint16_t *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;
    uint64_t n_tokens;
    uint32_t lanes_per_row, tokens_per_item;
    const int64_t* slots;

    BAM_DEV uint32_t counters(uint32_t) const { return 0; }

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        const uint32_t lane = threadIdx.x & 31u;
        const uint64_t warp = ((uint64_t)vb * blockDim.x + threadIdx.x) >> 5, nwarps = ((uint64_t)nvb * blockDim.x) >> 5;
        const uint32_t G = lanes_per_row, rows = 32u / G, c = lane & (G - 1u), grp = lane / G;
        const bool in_row = c < L.chunks;
        if (status_bad(L.r.cache.status)) return;
        const uint64_t groups = (n_tokens + tokens_per_item - 1) / tokens_per_item;
        for (uint64_t it = warp; it < groups * L.n_kv_heads; it = nwarps + L.draw()) {
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
                for (uint32_t i0 = 0; i0 < tokens_per_item; i0 += rows * KV_ROWS_AHEAD) {
                    uint4 kk[KV_ROWS_AHEAD], vv[KV_ROWS_AHEAD];
#pragma unroll
                    for (int e = 0; e < KV_ROWS_AHEAD; e++) {
                        const uint32_t i = i0 + e * rows, src = (i + grp) & 31u;
                        const uint64_t base = __shfl_sync(0xffffffffu, addr, src);
                        const uint32_t rr = __shfl_sync(0xffffffffu, row, src);
                        kk[e] = vv[e] = make_uint4(0, 0, 0, 0);
                        if (in_row && i + grp < tokens_per_item && ((m >> src) & 1u) && base) {
                            /* past L1: a slot can hold another page now than earlier in this launch */
                            const uint8_t* p = reinterpret_cast<const uint8_t*>(base) + rr * L.row_bytes() + L.swizzle(rr, c) * 16u;
                            kk[e] = ld_cg_v4(p);
                            vv[e] = ld_cg_v4(p + L.v_offset());
                        }
                    }
#pragma unroll
                    for (int e = 0; e < KV_ROWS_AHEAD; e++) {
                        const uint32_t i = i0 + e * rows, src = (i + grp) & 31u;
                        if (in_row && i + grp < tokens_per_item && ((m >> src) & 1u)) {
                            kv_store8(k + (int64_t)(t0 + src) * k_st + h * k_sh + c * 8, kk[e], VEC);
                            kv_store8(v + (int64_t)(t0 + src) * v_st + h * v_sh + c * 8, vv[e], VEC);
                        }
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

/* what a launch would fault on */
bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

bool on_16(const void* p, int64_t s0, int64_t s1) { return ((uintptr_t)p & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0; }

/* tokens a warp takes at a time: as many (up to `most`) as still make an item for every warp */
uint32_t tokens_of_item(uint64_t n_tokens, uint32_t parts, uint64_t warps, uint32_t most)
{
    uint32_t t = most;
    while (t > 1 && (n_tokens + t - 1) / t * parts < warps) t >>= 1;
    return t;
}

/* heads a warp takes at a time: as many (`least` to `most`) as still make `enough` items of so many pieces */
uint32_t heads_of_item(uint32_t heads, uint64_t pieces, uint64_t enough, uint32_t most, uint32_t least)
{
    uint32_t h = most;
    while (h > least && pieces * ((heads + h - 1) / h) < enough) h >>= 1;
    return h;
}

}  // namespace

extern "C" uint64_t bam_kv_scratch_bytes(bam_array_t a, const bam_kv_layout_t* layout)
{
    kv_layout_d_t L;
    if (kv_layout(a, layout, &L) != BAM_OK) return 0;
    const uint32_t most = kv_most_blocks(a);
    return kv_parts_at(most * KV_WORKERS) + (uint64_t)most * KV_WORKERS * 2 * KV_ROWS * (L.head_dim + 2) * sizeof(float);
}

extern "C" int bam_kv_scratch_init(bam_array_t a, void* scratch_dev, uint64_t scratch_bytes, void* stream)
{
    if (!a || !scratch_dev || ((uintptr_t)scratch_dev & 127)) return BAM_EINVAL;
    const uint64_t head = kv_parts_at(kv_most_blocks(a) * KV_WORKERS);
    if (scratch_bytes < head) return BAM_EINVAL;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    CK(cudaMemsetAsync(scratch_dev, 0xff, head, (cudaStream_t)stream));
    return BAM_OK;
}

extern "C" uint64_t bam_kv_stream_id(void* stream)
{
    unsigned long long id = 0;
    if (cudaStreamGetId((cudaStream_t)stream, &id) == cudaSuccess) return id;
    (void)cudaGetLastError();
    return ~0ull;
}

static int check_scratch(bam_array_t a, const bam_kv_layout_t* layout, void* scratch, uint64_t scratch_bytes)
{
    if (!scratch || ((uintptr_t)scratch & 127)) return BAM_EINVAL;
    return scratch_bytes < bam_kv_scratch_bytes(a, layout) ? BAM_EINVAL : BAM_OK;
}

template <class T, bool VEC>
static int launch_append_as(bam_array_t a, const kv_layout_d_t& L, const bam_kv_append_t* p, void* scratch, void* stream)
{
    KvAppendWork<T, VEC> w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.q = (const uint16_t*)p->q; w.k = (const uint16_t*)p->k; w.v = (const uint16_t*)p->v; w.q_out = (uint16_t*)p->q_out;
    w.q_st = p->q_stride[0]; w.q_sh = p->q_stride[1]; w.k_st = p->k_stride[0]; w.k_sh = p->k_stride[1];
    w.v_st = p->v_stride[0]; w.v_sh = p->v_stride[1]; w.qo_st = p->q_out_stride[0]; w.qo_sh = p->q_out_stride[1];
    w.n_tokens = p->n_tokens; w.n_q_heads = p->q ? p->n_q_heads : 0;
    w.lanes_per_row = lanes_of_row(L.chunks / 2);
    const uint64_t warps = (uint64_t)a->pc->ctrl->num_sms * w.min_blocks * (w.threads / 32);
    w.k_heads = heads_of_item(L.n_kv_heads, p->n_tokens / L.block_tokens, warps / 4, 4, 1);
    w.q_heads = heads_of_item(w.n_q_heads, p->n_tokens, 2 * warps, 32, 16);
    w.k_parts = (L.n_kv_heads + w.k_heads - 1) / w.k_heads;
    w.q_parts = (w.n_q_heads + w.q_heads - 1) / w.q_heads;
    w.k_tokens = tokens_of_item(p->n_tokens, w.k_parts, warps, KV_MAX_LANE_TOKENS);
    w.q_tokens = tokens_of_item(p->n_tokens, w.q_parts, 2 * warps, 16);
    w.slots = p->slots;
    w.rope.positions = p->positions; w.rope.cos = p->cos; w.rope.sin = p->sin; w.rope.n_positions = p->n_positions;
    w.rope.stride = p->rope_stride; w.rope.rotary_dim = p->cos ? p->rotary_dim : 0; w.rope.style = p->rope_style;
    w.q_norm = (const uint16_t*)p->q_norm; w.k_norm = (const uint16_t*)p->k_norm; w.eps = p->norm_eps; w.inv_dim = 1.f / (float)L.head_dim;
    const uint64_t items = (p->n_tokens + w.k_tokens - 1) / w.k_tokens * w.k_parts + (p->n_tokens + w.q_tokens - 1) / w.q_tokens * w.q_parts;
    return kv_launch(a->pc->ctrl, w, items, scratch, (cudaStream_t)stream);
}

template <class T>
static int launch_append(bam_array_t a, const kv_layout_d_t& L, const bam_kv_append_t* p, void* scratch, void* stream)
{
    const bool vec = (!p->q || (on_16(p->q, p->q_stride[0], p->q_stride[1]) && on_16(p->q_out, p->q_out_stride[0], p->q_out_stride[1]))) &&
                     on_16(p->k, p->k_stride[0], p->k_stride[1]) && on_16(p->v, p->v_stride[0], p->v_stride[1]) && on_16(p->q_norm, 0, 0) &&
                     on_16(p->k_norm, 0, 0) && on_16(p->cos, 2 * p->rope_stride, 0) && on_16(p->sin, 2 * p->rope_stride, 0);
    return vec ? launch_append_as<T, true>(a, L, p, scratch, stream) : launch_append_as<T, false>(a, L, p, scratch, stream);
}

extern "C" int bam_launch_kv_append(bam_array_t a, const bam_kv_layout_t* layout, const bam_kv_append_t* p, void* scratch_dev,
                                    uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!p || !p->k || !p->v || !p->slots || p->n_tokens > 0x7fffffffull) return BAM_EINVAL;
    if (!aligned(p->q, 2) || !aligned(p->k, 2) || !aligned(p->v, 2) || !aligned(p->q_out, 2) || !aligned(p->q_norm, 2) || !aligned(p->k_norm, 2) ||
        !aligned(p->slots, 8) || !aligned(p->positions, 8) || !aligned(p->cos, 4) || !aligned(p->sin, 4)) return BAM_EINVAL;
    if (p->q && (!p->q_out || p->n_q_heads == 0 || p->n_q_heads > 65536)) return BAM_EINVAL;
    if (p->cos || p->sin) {
        if (!p->cos || !p->sin || !p->positions || p->n_positions == 0 || p->n_positions > 0x7fffffffffffull) return BAM_EINVAL;
        if (p->rotary_dim == 0 || p->rotary_dim > L.head_dim || p->rotary_dim % 16 || p->rope_stride < 0) return BAM_EINVAL;
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

template <bool VEC>
static int launch_gather(bam_array_t a, const kv_layout_d_t& L, uint64_t n_tokens, const int64_t* slots_dev, void* k_out_dev, void* v_out_dev,
                         const int64_t* k_stride, const int64_t* v_stride, void* scratch, void* stream)
{
    KvGatherWork<VEC> w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.k = (uint16_t*)k_out_dev; w.v = (uint16_t*)v_out_dev;
    w.k_st = k_stride[0]; w.k_sh = k_stride[1]; w.v_st = v_stride[0]; w.v_sh = v_stride[1];
    w.n_tokens = n_tokens;
    w.lanes_per_row = lanes_of_row(L.chunks);
    const uint64_t warps = (uint64_t)a->pc->ctrl->num_sms * w.min_blocks * (w.threads / 32);
    w.tokens_per_item = tokens_of_item(n_tokens, L.n_kv_heads, warps, KV_MAX_LANE_TOKENS);
    w.slots = slots_dev;
    const uint64_t items = (n_tokens + w.tokens_per_item - 1) / w.tokens_per_item * L.n_kv_heads;
    return kv_launch(a->pc->ctrl, w, items, scratch, (cudaStream_t)stream);
}

extern "C" int bam_launch_kv_gather(bam_array_t a, const bam_kv_layout_t* layout, uint64_t n_tokens, const int64_t* slots_dev,
                                    void* k_out_dev, void* v_out_dev, const int64_t* k_stride, const int64_t* v_stride,
                                    void* scratch_dev, uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!slots_dev || !k_out_dev || !v_out_dev || !k_stride || !v_stride || n_tokens > 0x7fffffffull) return BAM_EINVAL;
    if (!aligned(slots_dev, 8) || !aligned(k_out_dev, 2) || !aligned(v_out_dev, 2)) return BAM_EINVAL;
    rc = check_scratch(a, layout, scratch_dev, scratch_bytes);
    if (rc) return rc;
    if (n_tokens == 0) return BAM_OK;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    const bool vec = on_16(k_out_dev, k_stride[0], k_stride[1]) && on_16(v_out_dev, v_stride[0], v_stride[1]);
    return vec ? launch_gather<true>(a, L, n_tokens, slots_dev, k_out_dev, v_out_dev, k_stride, v_stride, scratch_dev, stream)
               : launch_gather<false>(a, L, n_tokens, slots_dev, k_out_dev, v_out_dev, k_stride, v_stride, scratch_dev, stream);
}

extern "C" int bam_launch_kv_attend(bam_array_t a, const bam_kv_layout_t* layout, const bam_kv_attend_t* p, void* scratch_dev,
                                    uint64_t scratch_bytes, void* stream)
{
    kv_layout_d_t L;
    int rc = kv_layout(a, layout, &L);
    if (rc) return rc;
    if (!p || !p->q || !p->out || !p->block_table || !p->seq_lens) return BAM_EINVAL;
    if (!aligned(p->q, 2) || !aligned(p->out, 2) || !aligned(p->lse, 4) || !aligned(p->block_table, 4) || !aligned(p->seq_lens, 4)) return BAM_EINVAL;
    if (p->n_q_heads == 0 || p->n_q_heads > 65536 || p->n_q_heads % L.n_kv_heads) return BAM_EINVAL;
    if (p->batch > (1u << 20) || p->table_width == 0 || p->table_width > (1u << 27) || p->window < 0 || p->sinks < 0) return BAM_EINVAL;
    if (!std::isfinite(p->scale)) return BAM_EINVAL;
    rc = check_scratch(a, layout, scratch_dev, scratch_bytes);
    if (rc) return rc;
    if (p->batch == 0) return BAM_OK;
    device_guard g;
    CK(g.enter(a->pc->ctrl->device));
    return layout->dtype == BAM_KV_BF16 ? kv_launch_attend<__nv_bfloat16>(a, L, p, scratch_dev, stream)
                                        : kv_launch_attend<__half>(a, L, p, scratch_dev, stream);
}
