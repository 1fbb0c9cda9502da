/*
 * bam_kv_attend.cuh -- attention of one new token per sequence over the key/value rows of bam_kv.cuh.
 */
#ifndef BAM_KV_ATTEND_CUH
#define BAM_KV_ATTEND_CUH

#include <cstring>

#include "bam_kv.cuh"

namespace bam {

/* The flattened work list: sequence b has `n` chunks of CS tokens with something visible in them, in each of its
 * n_kv_heads * tiles units (a unit: 16 query heads of one key/value head), and the list is b-major, then unit, then
 * chunk.  Worker block i takes the chunks [i * per, (i + 1) * per): every block reads the same amount whatever the
 * lengths are, a long sequence is split over many blocks and a short one is not split at all.  A block that does not
 * own a whole unit writes its running maximum, denominator and unnormalised sum to the scratch; the blocks of a unit
 * wait for each other at the end (they are co-resident, one cooperative launch) and each joins a part of the output,
 * adding in a fixed order: the same bits on every run.
 *
 * What bounds it is reading keys and values once from HBM: 4 head_dim bytes a token for 4 head_dim flops a query head,
 * 8 flops a byte at 8 query heads.  So the design feeds bulk copies.  One warp looks pages up and pins them, 32 at a
 * time, up to 64 chunks ahead: a look-up is a chain of six dependent accesses that miss L2 while the rows stream
 * through it, 5 to 10 us.  Three consumer warps take the chunks in turn; each has its own stages of shared memory
 * and refills them itself, keys and values with one bulk copy each, so no warp waits for another between units.  A
 * page is unpinned as soon as its rows have landed.  Every warp keeps one running softmax, merged once per unit.
 * The products go through m16n8k16 matrix instructions (8.3 cycles each per quarter SM, measured): 16 query heads are
 * all the rows there are, and a chunk of 32 tokens at 128 dimensions takes 200 of the 710 cycles that HBM needs to
 * deliver it to an SM; the 128-row tcgen05 tiles would be seven eighths padding. */
#define KV_STAGES_MAX 24u
#define KV_AHEAD 64u                  /* chunks whose pages may be pinned at a time, in batches of 32 */
#define KV_CONSUMERS 3u               /* consumer warps: with the pinning warp four, which leaves a thread 255 registers */
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
template <uint32_t N> BAM_DEV void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N * 32) : "memory"); }
/* 2^x, off by two units in the last place at most; results below the normal range are 0 */
BAM_DEV float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
BAM_DEV void st_cg_f4(float* p, float x, float y, float z, float w)
{
    asm volatile("st.global.cg.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
BAM_DEV void st_cg_f2(float* p, float x, float y) { asm volatile("st.global.cg.v2.f32 [%0], {%1,%2};" ::"l"(p), "f"(x), "f"(y) : "memory"); }
BAM_DEV float ld_cg_f(const float* p) { float v; asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory"); return v; }

/* A pinned chunk: where its rows are.  `tag` is 2 r while the place is free for its r-th chunk and 2 r + 1 from the
 * moment that chunk is pinned until it is unpinned. */
struct kv_pinned_t {
    uint64_t src;
    uint32_t slot, rows;              /* rows: first row in the stage << 16 | number of rows; 0: the block was no block */
};

/* Shared memory of a worker block behind its ring of stages. */
template <int DMAX>
struct kv_shared_t {
    float merge[KV_ROWS][DMAX < 128 ? DMAX : 128];      /* a warp's sums on their way into another's   */
    float m[KV_CONSUMERS][KV_ROWS], l[KV_CONSUMERS][KV_ROWS];
    uint64_t full[KV_STAGES_MAX];
    kv_pinned_t pinned[KV_AHEAD];
    uint32_t tag[KV_AHEAD];
    uint64_t warp_sum[8];
    uint64_t start_pos;
    uint32_t start_b;
    volatile uint32_t abort;
    struct { uint32_t b, u; uint64_t first; uint32_t n; } join[2];
};

BAM_DEV uint32_t ld_acquire_cta(const uint32_t* p) { uint32_t v; asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory"); return v; }
BAM_DEV void st_release_cta(uint32_t* p, uint32_t v) { asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory"); }

/* DMAX: the head_dim the registers are laid out for, and with EXACT the head_dim itself (otherwise every step over
 * the dimensions asks whether it is needed, which keeps the compiler from overlapping them: 3 times the time of a
 * chunk at 128); CS: tokens of a chunk (it divides block_tokens). */
template <class T, int DMAX, int CS, bool EXACT>
struct KvAttendWork {
    static constexpr uint32_t CONSUMERS = KV_CONSUMERS;
    typedef kv_shared_t<DMAX> shared_t;
    static constexpr int threads = 32 * (CONSUMERS + 1), min_blocks = 2;
    static constexpr uint32_t smem = 112 * 1024;
    static constexpr uint32_t ring_bytes = (smem - 1024u - (uint32_t)sizeof(shared_t)) & ~1023u;
    static constexpr bool pow2_row = EXACT && (DMAX == 64 || DMAX == 128 || DMAX == 256);
    kv_layout_d_t L;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    int64_t q_sb, q_sh, o_sb, o_sh, table_stride;
    const int32_t *table, *lens;
    uint32_t batch, n_q_heads, table_width;
    uint32_t q32, o32;                                   /* two elements at a time lie on 4-byte boundaries */
    uint32_t group, tiles;                               /* query heads of a key/value head, units they make */
    float scale_log2;                                    /* its magnitude; the sign goes into the query */
    uint32_t q_sign;
    int64_t window, sinks;
    uint32_t* arrived;                                   /* per worker block, all ones at the start: arrivals at the unit it begins */
    float* parts;                                        /* [worker block][2]: head_dim x 16 sums, 16 maxima, 16 denominators */

    BAM_DEV uint32_t dim() const { return EXACT ? (uint32_t)DMAX : L.head_dim; }
    BAM_DEV uint32_t row_bytes() const { return dim() * 2u; }
    BAM_DEV uint32_t stages() const
    {
        /* a multiple of the consumers: every stage then belongs to one warp, which meets its uses in order (a phase
         * of an mbarrier can only be told from the one before it) */
        const uint32_t n = ring_bytes / (CS * dim() * 4u);
        return (n < KV_STAGES_MAX ? n : KV_STAGES_MAX) / CONSUMERS * CONSUMERS;
    }
    BAM_DEV float* part(uint32_t block, uint32_t which) const { return parts + ((size_t)block * 2 + which) * (KV_ROWS * (dim() + 2)); }

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

    /* A warp's wait, and it ends: `done`, asked by all lanes together, says when; false when the block gives up
     * (someone's wait ran out, or the status block says so). */
    template <class Done>
    BAM_DEV bool wait(shared_t& sh, Done done) const
    {
        uint32_t polls = 0;
        uint64_t t0 = 0;
        while (!done()) {
            bool stop = sh.abort;
            if (((++polls) & 255u) == 0u) {
                bam_status_t* st = L.r.cache.status;
                const uint64_t now = global_timer_ns();
                if (t0 == 0) t0 = now;
                /* the pinning warp's own waits have one limit each; twice that is more than it needs to report */
                if (now - t0 > 2 * st->spin_timeout_ns) status_fail(st, BAM_ETIMEDOUT, BAM_AT_TMA, polls);
                stop |= status_bad(st);
            }
            if (__any_sync(0xffffffffu, stop)) { sh.abort = 1; return false; }
        }
        return true;
    }

    /* ---- the pinning warp ------------------------------------------------------------------------------ */
    BAM_DEV void pin_ahead(shared_t& sh, uint64_t f0, uint64_t f1, uint32_t vb) const
    {
        const uint32_t full_mask = 0xffffffffu, lane = lane_id();
        const uint32_t units = L.n_kv_heads * tiles;
        uint32_t base_b = sh.start_b;
        uint64_t base_pos = sh.start_pos;
        spin_t sp;
        for (uint64_t f = f0; f < f1; f += 32) {
            bool pending = f + lane < f1;
            /* where this lane's chunk is */
            uint32_t b = base_b, rows = 0;
            uint64_t pos = base_pos + lane, page = 0, offset = 0;
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
                else {
                    page = L.page_of((uint64_t)block, u / tiles);
                    rows = (uint32_t)(lo - t0) << 16 | (uint32_t)(hi - lo);
                    offset = (uint64_t)(lo % L.block_tokens) * row_bytes();
                }
            }
            base_b = __shfl_sync(full_mask, b, 31);
            base_pos = __shfl_sync(full_mask, pos, 31) + 1;
            const uint32_t k = (uint32_t)(f - f0) + lane, place = k % KV_AHEAD, round = k / KV_AHEAD;
            if (!wait(sh, [&] { return __all_sync(full_mask, !pending || ld_acquire_cta(&sh.tag[place]) == 2u * round); })) return;
            /* A lane whose page cannot be had now is asked for again when
             * the chunks before it have been handed on, and the chunks behind it give theirs back meanwhile: what a
             * block holds is always the next it needs, so blocks never wait for pages that wait for them */
            sp.reset();
            uint32_t ask = 32;                 /* lanes that ask at a time: fewer in a cache that is too full for all, down to one */
            for (;;) {
                const uint32_t todo = __ballot_sync(full_mask, pending);
                if (todo == 0u) break;
                const uint32_t upto = __ffs(todo) - 1 + ask;
                const bool want = pending && !bad && lane < upto;
                const uint32_t slot = kv_pin_warp(L, want, page, false, vb * 8u);
                const bool got = want && slot <= BAM_SLOT_MAX;
                const uint32_t miss = __ballot_sync(full_mask, want && !got);
                const uint32_t last = miss ? __ffs(miss) - 1 : upto;               /* the lanes below go out now */
                ask = miss ? (ask + 1) / 2 : (ask < 32u ? ask * 2 : 32u);
                const bool failed = __any_sync(full_mask, want && slot == BAM_SLOT_ERR);
                if (got && (lane >= last || failed)) L.r.release_page(slot, 1);
                if (failed) { sh.abort = 1; return; }
                if (pending && lane < last) {
                    kv_pinned_t* e = &sh.pinned[place];
                    e->src = got ? L.r.get_cache_page_addr(slot) + offset : 0;
                    e->slot = got ? slot : BAM_SLOT_NONE;
                    e->rows = rows;
                    st_release_cta(&sh.tag[place], 2u * round + 1u);
                    pending = false;
                }
                if (__ballot_sync(full_mask, pending) == todo && __any_sync(full_mask, sp.expired(L.r.cache.status, BAM_AT_FIND_SLOT, page))) {
                    sh.abort = 1;
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
        a[0] = r0 ? q_pair(r0, d) ^ q_sign : 0u;
        a[1] = r1 ? q_pair(r1, d) ^ q_sign : 0u;
        a[2] = r0 ? q_pair(r0, d + 8) ^ q_sign : 0u;
        a[3] = r1 ? q_pair(r1, d + 8) ^ q_sign : 0u;
    }

    /* A consumer warp's own chunks of the block (w, w + CONSUMERS, ...) and its stages. */
    struct ring_t {
        uint32_t base, end;             /* shared address of the ring; chunks of the block                */
        uint32_t next, stage, use;      /* the chunk that is consumed next, its stage and how often that was used */
        uint32_t issue, issue_stage;    /* the chunk that is copied next                                  */
    };

    /* Start the copies of the warp's next chunk, if it has a free stage and the chunk is pinned; false if not.  Nothing
     * is waited for: what the warp holds pinned is what it consumes without anybody's help, so that blocks never wait
     * for pages that wait for them. */
    BAM_DEV bool issue_next(shared_t& sh, ring_t& g) const
    {
        if (g.issue >= g.end || g.issue - g.next >= stages()) return false;
        const uint32_t place = g.issue % KV_AHEAD, round = g.issue / KV_AHEAD;
        uint32_t ready = 0;
        if (lane_id() == 0) ready = ld_acquire_cta(&sh.tag[place]) == 2u * round + 1u ? 1u : 0u;
        if (!__shfl_sync(0xffffffffu, ready, 0)) return false;
        if (lane_id() == 0) {
            const kv_pinned_t e = sh.pinned[place];
            const uint32_t full = smem_u32(&sh.full[g.issue_stage]);
            if (e.slot == BAM_SLOT_NONE) mbar_arrive(full);
            else {
                const uint32_t bytes = (e.rows & 0xffffu) * row_bytes();
                const uint32_t dst = g.base + g.issue_stage * (CS * dim() * 4u) + (e.rows >> 16) * row_bytes();
                /* pages that this launch fetched were written by bulk copies too; order those before ours */
                asm volatile("fence.proxy.async.global;" ::: "memory");
                mbar_expect_tx(full, 2 * bytes);
                bulk_load(dst, reinterpret_cast<const void*>(e.src), bytes, full);
                bulk_load(dst + CS * row_bytes(), reinterpret_cast<const void*>(e.src + L.v_offset()), bytes, full);
            }
        }
        __syncwarp();
        g.issue += CONSUMERS;
        g.issue_stage += CONSUMERS;
        if (g.issue_stage >= stages()) g.issue_stage -= stages();
        return true;
    }
    /* Wait until the warp's next chunk has landed, and start copies of later ones meanwhile. */
    BAM_DEV bool landed(shared_t& sh, ring_t& g) const
    {
        const uint32_t full = smem_u32(&sh.full[g.stage]);
        return wait(sh, [&] {
            while (issue_next(sh, g)) {}
            return g.next < g.issue && __all_sync(0xffffffffu, mbar_test(full, g.use & 1u));
        });
    }
    /* The warp's next chunk has landed: unpin its page.  (Lane 0.)  The rows are in shared memory, nothing of this
     * thread is outstanding that a release would have to wait for; its fence held the warp up for 2000 cycles. */
    BAM_DEV void unpin(shared_t& sh, uint32_t n) const
    {
        const uint32_t place = n % KV_AHEAD, slot = sh.pinned[place].slot;
        if (slot != BAM_SLOT_NONE) red_add_relaxed(&L.r.cache.slots[slot].state, 0u - 1u);
        st_release_cta(&sh.tag[place], 2u * (n / KV_AHEAD) + 2u);
    }

    struct state_t {
        float o[DMAX / 8][4];
        float m[2], l[2];
    };

    /* One chunk: S = Q K^T, p = 2^(S scale log2(e) - m), O += p V.  The weights go into the product as two 16-bit
     * parts, p = hi + lo, which keeps 16 (bf16) or more bits of them: the product runs twice, on a pipe that idles. */
    template <bool WHOLE>
    BAM_DEV void chunk(state_t& z, const uint32_t (&qa)[DMAX / 16][4], uint32_t stage, const kv_seen_t& v, int64_t t0) const
    {
        const uint32_t lane = lane_id(), rb = row_bytes();
        const uint32_t x = pow2_row ? lane & 7u : ((lane & 7u) >> L.swz_shift) & L.swz_mask;
        /* 16-byte chunk c (even) + the lane's own bit of a row: where rows are powers of two and the stage is aligned
         * to them, one XOR */
        auto at = [&](uint32_t base, uint32_t own, uint32_t c) {
            return pow2_row ? (base + ((own ^ x) * 16u)) ^ (c * 16u) : base + ((c + own) ^ x) * 16u;
        };
        float s[CS / 8][4];
#pragma unroll
        for (int i = 0; i < CS / 8; i++) { s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f; }
        const uint32_t k_row = stage + ((lane & 7u) + ((lane >> 4) & 1u) * 8u) * rb, k_c = (lane >> 3) & 1u;
#pragma unroll
        for (int ks = 0; ks < DMAX / 16; ks++) {
            if (EXACT || ks * 16 < (int)L.head_dim) {
#pragma unroll
                for (int np = 0; np < CS / 16; np++) {
                    uint32_t r[4];
                    ldm_x4(r, at(k_row, k_c, ks * 2) + np * 16 * rb);
                    mma_16816(s[2 * np], qa[ks], r[0], r[1], T());
                    mma_16816(s[2 * np + 1], qa[ks], r[2], r[3], T());
                }
            }
        }
        /* bit i: this lane's column i (of its CS / 4) is visible */
        uint32_t vis = 0;
        if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < CS / 4; i++) {
                const int64_t j = t0 + (i >> 1) * 8 + (lane & 3u) * 2 + (i & 1);
                if ((j < v.first || j >= v.begin) && j < v.len) vis |= 1u << i;
            }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < CS / 8; i++) {
            if (!WHOLE) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (!((vis >> (2 * i + (e & 1))) & 1u)) s[i][e] = -INFINITY;
            }
            mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][1]));
            mx1 = fmaxf(mx1, fmaxf(s[i][2], s[i][3]));
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float n0 = fmaxf(z.m[0], mx0 * scale_log2), n1 = fmaxf(z.m[1], mx1 * scale_log2);
        const float c0 = n0 == -INFINITY ? 0.f : n0, c1 = n1 == -INFINITY ? 0.f : n1;     /* nothing seen yet: exp2(-inf - 0) = 0 */
        if (__any_sync(0xffffffffu, n0 != z.m[0] || n1 != z.m[1])) {
            const float a0 = exp2_fast(z.m[0] - c0), a1 = exp2_fast(z.m[1] - c1);
            z.l[0] *= a0; z.l[1] *= a1;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) { z.o[i][0] *= a0; z.o[i][1] *= a0; z.o[i][2] *= a1; z.o[i][3] *= a1; }
            z.m[0] = n0; z.m[1] = n1;
        }
        const uint32_t v_row = stage + CS * rb + ((lane & 7u) + ((lane >> 3) & 1u) * 8u) * rb, v_c = (lane >> 4) & 1u;
        uint32_t hi[CS / 16][4], lo[CS / 16][4];
#pragma unroll
        for (int i = 0; i < CS / 8; i++) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[e] = exp2_fast(fmaf(s[i][e], scale_log2, e < 2 ? -c0 : -c1));
                if (!WHOLE && !((vis >> (2 * i + (e & 1))) & 1u)) p[e] = 0.f;
            }
            z.l[0] += p[0] + p[1];
            z.l[1] += p[2] + p[3];
            uint32_t* h = hi[i / 2] + 2 * (i & 1);
            uint32_t* l = lo[i / 2] + 2 * (i & 1);
            h[0] = kv_type<T>::pack(p[0], p[1]);
            h[1] = kv_type<T>::pack(p[2], p[3]);
            const float2 h0 = kv_type<T>::unpack(h[0]), h1 = kv_type<T>::unpack(h[1]);
            l[0] = kv_type<T>::pack(p[0] - h0.x, p[1] - h0.y);
            l[1] = kv_type<T>::pack(p[2] - h1.x, p[3] - h1.y);
        }
#pragma unroll
        for (int kt = 0; kt < CS / 16; kt++) {
            /* rows that are not visible may hold anything, and 0 x NaN is not 0: they become zeros */
            uint32_t k0 = 0, k1 = 0;
            if (!WHOLE) {
                const uint32_t bits = vis >> (4 * kt);
                k0 = ((bits & 1u) ? 0x0000ffffu : 0u) | ((bits & 2u) ? 0xffff0000u : 0u);
                k1 = ((bits & 4u) ? 0x0000ffffu : 0u) | ((bits & 8u) ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int np = 0; np < DMAX / 16; np++) {
                if (EXACT || np * 16 < (int)L.head_dim) {
                    uint32_t r[4];
                    ldm_x4_t(r, at(v_row, v_c, np * 2) + kt * 16 * rb);
                    if (!WHOLE) { r[0] &= k0; r[1] &= k1; r[2] &= k0; r[3] &= k1; }
                    mma_16816(z.o[2 * np], hi[kt], r[0], r[1], T());
                    mma_16816(z.o[2 * np + 1], hi[kt], r[2], r[3], T());
                    mma_16816(z.o[2 * np], lo[kt], r[0], r[1], T());
                    mma_16816(z.o[2 * np + 1], lo[kt], r[2], r[3], T());
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
                    if (i * 8 < (int)L.head_dim || EXACT) store_pair(p + i * 8, z.o[i][2 * half] * inv, z.o[i][2 * half + 1] * inv);
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
            float* row = p + r * dim() + (lane & 3u) * 2;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++)
                if (i * 8 < (int)L.head_dim || EXACT) st_cg_f2(row + i * 8, z.o[i][2 * half], z.o[i][2 * half + 1]);
            if ((lane & 3u) == 0u) {
                float* ml = p + KV_ROWS * dim();
                ml[r] = z.m[half];
                ml[KV_ROWS + r] = z.l[half];
            }
        }
    }

    /* Merge the consumers' states into warp 0's. */
    BAM_DEV void merge(shared_t& sh, state_t& z, uint32_t w) const
    {
        const uint32_t lane = lane_id(), row = lane >> 2;
        if ((lane & 3u) == 0u) {
#pragma unroll
            for (int half = 0; half < 2; half++) { sh.m[w][row + 8 * half] = z.m[half]; sh.l[w][row + 8 * half] = z.l[half]; }
        }
        consumers_sync<CONSUMERS>();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = row + 8 * half;
            float M = -INFINITY, l = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < CONSUMERS; k++) M = fmaxf(M, sh.m[k][r]);
            const float c = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (uint32_t k = 0; k < CONSUMERS; k++) l += sh.l[k][r] * exp2_fast(sh.m[k][r] - c);
            const float a = exp2_fast(z.m[half] - c);
            z.m[half] = M;
            z.l[half] = l;
#pragma unroll
            for (int i = 0; i < DMAX / 8; i++) { z.o[i][2 * half] *= a; z.o[i][2 * half + 1] *= a; }
        }
        /* warp 2's sums into warp 1's, those into warp 0's, through one buffer of up to 128 dimensions at a time */
        constexpr int W = DMAX < 128 ? DMAX : 128;
#pragma unroll
        for (int d0 = 0; d0 < DMAX; d0 += W) {
            auto move = [&](bool in) {
#pragma unroll
                for (int i = d0 / 8; i < (d0 + W) / 8; i++) {
                    if (i * 8 < DMAX && (EXACT || i * 8 < (int)L.head_dim)) {
                        float2* p = reinterpret_cast<float2*>(&sh.merge[row][i * 8 - d0 + (lane & 3u) * 2]);
                        float2* q8 = reinterpret_cast<float2*>(&sh.merge[row + 8][i * 8 - d0 + (lane & 3u) * 2]);
                        if (in) { z.o[i][0] += p->x; z.o[i][1] += p->y; z.o[i][2] += q8->x; z.o[i][3] += q8->y; }
                        else { *p = make_float2(z.o[i][0], z.o[i][1]); *q8 = make_float2(z.o[i][2], z.o[i][3]); }
                    }
                }
            };
            static_assert(CONSUMERS == 3, "the chain below");
            if (w == 2) move(false);
            consumers_sync<CONSUMERS>();
            if (w == 1) { move(true); move(false); }          /* a thread writes where it has read */
            consumers_sync<CONSUMERS>();
            if (w == 0) move(true);
            consumers_sync<CONSUMERS>();
        }
    }

    BAM_DEV void consume(shared_t& sh, uint32_t ring, uint64_t f0, uint64_t f1, uint64_t per, uint32_t vb) const
    {
        const uint32_t lane = lane_id(), w = threadIdx.x >> 5;
        const uint32_t S = stages(), stage_bytes = CS * dim() * 4u, units = L.n_kv_heads * tiles;
        uint32_t b = sh.start_b, n_join = 0;
        uint64_t pos = sh.start_pos;
        ring_t g = { ring, (uint32_t)(f1 - f0), w, w, 0, w, w };
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
            uint32_t qa[DMAX / 16][4];
            const uint32_t mine = (w + CONSUMERS - (uint32_t)((f - f0) % CONSUMERS)) % CONSUMERS;      /* first chunk of the segment that is this warp's */
            if (mine < seg) {
#pragma unroll
                for (int ks = 0; ks < DMAX / 16; ks++)
                    if (EXACT || ks * 16 < (int)L.head_dim) load_q(qa[ks], q0, q1, ks);
            }
            for (uint32_t i = mine; i < seg; i += CONSUMERS) {
                if (!landed(sh, g)) continue;
                const bool there = sh.pinned[g.next % KV_AHEAD].slot != BAM_SLOT_NONE;
                __syncwarp();
                if (lane == 0) unpin(sh, g.next);
                if (there) {
                    const int64_t t0 = first_token(v, c + i);
                    if (t0 + CS <= v.first || (t0 >= v.begin && t0 + CS <= v.len)) chunk<true>(z, qa, ring + g.stage * stage_bytes, v, t0);
                    else chunk<false>(z, qa, ring + g.stage * stage_bytes, v, t0);
                }
                __syncwarp();
                g.next += CONSUMERS;
                g.stage += CONSUMERS;
                if (g.stage >= S) { g.stage -= S; g.use++; }
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
        /* given up: copies that are still under way land (bounded) before the block leaves */
        while (g.next < g.issue) {
            const uint64_t since = global_timer_ns();
            const uint32_t full = smem_u32(&sh.full[g.stage]);
            while (!mbar_test(full, g.use & 1u) && global_timer_ns() - since < 2 * L.r.cache.status->spin_timeout_ns) {}
            __syncwarp();
            if (lane == 0) unpin(sh, g.next);
            g.next += CONSUMERS;
            g.stage += CONSUMERS;
            if (g.stage >= S) { g.stage -= S; g.use++; }
        }
        consumers_sync<CONSUMERS>();
        for (uint32_t k = 0; k < n_join; k++) join(sh, sh.join[k].b, sh.join[k].u, sh.join[k].first, sh.join[k].n, per, vb);
    }

    /* This block's share of a unit that several blocks worked on. */
    BAM_DEV void join(shared_t& sh, uint32_t b, uint32_t u, uint64_t U0, uint32_t n, uint64_t per, uint32_t vb) const
    {
        const uint32_t lane = lane_id(), w = threadIdx.x >> 5, D = dim();
        const uint32_t i0 = (uint32_t)(U0 / per), cnt = (uint32_t)((U0 + n - 1) / per) - i0 + 1, j = vb - i0;
        if (threadIdx.x == 0) {
            spin_t sp;
            while (ld_acquire_gpu(arrived + i0) != cnt - 1u) {
                if (sh.abort) break;
                if (sp.expired(L.r.cache.status, BAM_AT_KV_JOIN, i0)) { sh.abort = 1; break; }
            }
        }
        consumers_sync<CONSUMERS>();
        if (__any_sync(0xffffffffu, sh.abort)) return;
        const uint32_t h = u / tiles, r0 = (u - h * tiles) * KV_ROWS;
        const uint32_t rows = group - r0 < KV_ROWS ? group - r0 : KV_ROWS, quads = rows * (D / 4);
        const uint32_t g0 = (uint32_t)((uint64_t)quads * j / cnt), g1 = (uint32_t)((uint64_t)quads * (j + 1) / cnt);
        uint32_t P = 1;
        while (P < cnt && P < 32u) P <<= 1;
        const uint32_t p = lane & (P - 1u), at_once = 32u / P * CONSUMERS;
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
                const float a = exp2_fast(ld_cg_f(q_ + KV_ROWS * D + r) - c);
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
        /* stages on 1 KB boundaries: the addresses within one are formed with XOR */
        uint8_t* const mem = bam_dyn_smem + (0u - smem_u32(bam_dyn_smem)) % 1024u;
        shared_t& sh = *reinterpret_cast<shared_t*>(mem + ring_bytes);
        const uint32_t ring = smem_u32(mem), t = threadIdx.x, lane = t & 31u, w = t >> 5;
        const uint32_t units = L.n_kv_heads * tiles, S = stages();
        if (t < S) {
            mbar_init(smem_u32(&sh.full[t]), 1);
        }
        if (t < KV_AHEAD) sh.tag[t] = 0;
        if (t == 0) sh.abort = status_bad(L.r.cache.status) ? 1u : 0u;
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
        for (uint32_t k = 0; k < CONSUMERS + 1; k++) {
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
            if (w == CONSUMERS) pin_ahead(sh, f0, f1, vb);
            else consume(sh, ring, f0, f1, per, vb);
        }
        __syncthreads();
        /* given up: pages that were pinned and never copied */
        if (sh.abort && t < KV_AHEAD && (sh.tag[t] & 1u) && sh.pinned[t].slot != BAM_SLOT_NONE) L.r.release_page(sh.pinned[t].slot, 1);
    }
};

template <class T, int DMAX, int CS, bool EXACT>
static int launch_attend_as(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    typedef KvAttendWork<T, DMAX, CS, EXACT> Work;
    Work w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.q = (const uint16_t*)p->q; w.out = (uint16_t*)p->out; w.lse = p->lse;
    w.q_sb = p->q_stride[0]; w.q_sh = p->q_stride[1]; w.o_sb = p->out_stride[0]; w.o_sh = p->out_stride[1];
    w.table = p->block_table; w.table_stride = p->table_stride; w.table_width = p->table_width; w.lens = p->seq_lens;
    w.batch = p->batch; w.n_q_heads = p->n_q_heads;
    w.group = p->n_q_heads / L.n_kv_heads; w.tiles = (w.group + KV_ROWS - 1) / KV_ROWS;
    w.scale_log2 = fabsf(p->scale) * 1.4426950408889634f;
    w.q_sign = p->scale < 0.f ? 0x80008000u : 0u;
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
int kv_launch_attend(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    /* chunks of 32 tokens halve what a chunk costs beside its products (softmax statistics, barriers); blocks that they
     * do not divide, and wide heads, whose registers are taken, go in chunks of 16 */
    const bool by32 = L.block_tokens % 32 == 0;
    switch (L.head_dim) {
    case 64: return by32 ? launch_attend_as<T, 64, 32, true>(a, L, p, scratch, stream) : launch_attend_as<T, 64, 16, true>(a, L, p, scratch, stream);
    case 80: return launch_attend_as<T, 80, 16, true>(a, L, p, scratch, stream);
    case 96: return launch_attend_as<T, 96, 16, true>(a, L, p, scratch, stream);
    case 128: return by32 ? launch_attend_as<T, 128, 32, true>(a, L, p, scratch, stream) : launch_attend_as<T, 128, 16, true>(a, L, p, scratch, stream);
    case 256: return launch_attend_as<T, 256, 16, true>(a, L, p, scratch, stream);
    default: break;
    }
    if (L.head_dim < 128) return launch_attend_as<T, 128, 16, false>(a, L, p, scratch, stream);
    return launch_attend_as<T, 256, 16, false>(a, L, p, scratch, stream);
}

}  // namespace bam
#endif
