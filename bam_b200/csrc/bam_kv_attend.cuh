/*
 * bam_kv_attend.cuh -- attention of one new token per sequence over the key/value rows of bam_kv.cuh.
 */
#ifndef BAM_KV_ATTEND_CUH
#define BAM_KV_ATTEND_CUH

#include <cfloat>
#include <cstring>

#include "bam_kv.cuh"

namespace bam {

/* The flattened work list: sequence b has `n` chunks of CS tokens with something visible in them, in each of its
 * n_kv_heads * tiles units (a unit: 16 query heads of one key/value head), and the list is b-major, then unit, then
 * chunk.  A WARP is a worker: it takes one of as many equal runs as there are workers, copies their chunks into its
 * own stages of shared memory and keeps one running softmax.  Every warp reads the same amount whatever the lengths
 * are: a long sequence is split over many warps, short ones are as many to a warp.  Warps share nothing and wait for
 * nothing of one another until the end: one that does not own a whole unit writes its running maximum, denominator and
 * unnormalised sum to the scratch, and then the warps of that unit wait for each other (they are co-resident, one
 * cooperative launch) and each joins a part of the output, adding in a fixed order: the same bits on every run.
 *
 * What bounds it is reading keys and values once from HBM: 4 head_dim bytes a token for 4 head_dim flops a query head,
 * 8 flops a byte at 8 query heads.  So the design feeds bulk copies: three worker warps a block, two blocks an SM, two
 * or more chunks under way for each (200 KB of an SM's shared memory).  The fourth warp of a block looks their pages
 * up and pins them up to 16 chunks ahead: a look-up is three dependent accesses that miss L2 while the rows stream
 * through it, 2 to 5 us (done by the workers themselves, 32 pages at a time, it cost 3 us of 186, and registers that
 * wide heads lack: 16 heads of 256 spill 32 to 44 bytes a thread as it is).  The products go through m16n8k16 matrix
 * instructions (8.3 cycles each per quarter SM, measured): up to 16 query heads are all there is, tcgen05 tiles of 64 or 128
 * rows would be mostly padding.  The scores have the queries as rows and the sums as columns, S = Q K^T and O^T = V^T P^T: the scores are then where the second
 * product wants its right operand, and eight query heads take half of the instructions (and of the registers for O)
 * that sixteen do.  At 128 dimensions a chunk of 32 tokens takes 64 of them, 130 of the 710 cycles that HBM needs to
 * deliver it to an SM.
 *
 * Measured (bf16, 8 key/value heads of 128): 64 sequences of 2500 to 4100 tokens, 867 MB, 165 us = 5.2 TB/s, 0.80 of a copy;
 * 32 of 130 to 1700, 120 MB, 47 us.  Time stamps of the latter's 744 workers, in us from the start of the first block: the list
 * is laid out at 2.5; the first chunk has landed at 9.5 (mean; 16.6 the last); the last of 11 chunks is consumed at 26.1 (21.3
 * to 34.3); the parts are written at 27.3 and joined at 33.9 (the last at 41.9); 5 more are the start of a cooperative launch
 * and the end of the controller blocks.  In the large case the workers' last chunks lie between 112 and 152 us: equal runs do
 * not end together.  A call costs the host 13 us. */
#define KV_STAGES_MAX 8u              /* stages of a worker */
#define KV_AHEAD 16u                  /* chunks of a worker that are pinned and not yet consumed, at most */
#define KV_PIN_LANES 10u              /* lanes of the pinning warp for each worker */
#define KV_MIN_CHUNKS 4u              /* a worker takes at least so many: 38 us with a window of 1024 in 48 sequences, 38.7 with 2,
                                       * 39.6 with 8 */

struct kv_seen_t {
    uint32_t len, first, begin;       /* visible: j < first, and begin <= j < len (lengths are 32-bit and positive) */
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
/* 2^x, off by two units in the last place at most; results below the normal range are 0 */
BAM_DEV float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
BAM_DEV void st_cg_f4(float* p, float x, float y, float z, float w)
{
    asm volatile("st.global.cg.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
BAM_DEV void st_cg_f2(float* p, float x, float y) { asm volatile("st.global.cg.v2.f32 [%0], {%1,%2};" ::"l"(p), "f"(x), "f"(y) : "memory"); }

/* Where a worker's run begins, or a chunk is: sequence, chunk within the sequence's share of the list. */
struct kv_place_t {
    uint64_t f, pos;
    uint32_t b;
};

/* A pinned chunk: where the rows of its pieces are.  `rows`: first row in the stage << 16 | number of rows. */
struct kv_pinned_t {
    uint64_t src[2];
    uint32_t slot[2], rows[2];
};

/* Shared memory of a worker block behind its stages. */
struct kv_shared_t {
    uint64_t full[KV_WORKERS][KV_STAGES_MAX];
    kv_pinned_t pinned[KV_WORKERS][KV_AHEAD];           /* chunk k of a worker at place k % ahead     */
    uint32_t tag[KV_WORKERS][KV_AHEAD];                 /* 2 r: free for its r-th chunk, 2 r + 1: from then on until that is unpinned */
    kv_place_t from[KV_WORKERS];                        /* where the workers' runs begin              */
    uint32_t chunks[KV_WORKERS];                        /* and how long they are                      */
    uint64_t before[32 * (KV_WORKERS + 1) + 1];         /* chunks of the list before each thread's run of sequences */
    uint64_t warp_sum[KV_WORKERS + 1];
    uint32_t warp_max[KV_WORKERS + 1];
    volatile uint32_t abort;
    struct { uint32_t b, u, first, workers; } join[KV_WORKERS][2];      /* units to be joined, by whom */
};

BAM_DEV uint32_t ld_acquire_cta(const uint32_t* p) { uint32_t v; asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory"); return v; }
BAM_DEV void st_release_cta(uint32_t* p, uint32_t v) { asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory"); }

/* DMAX: the head_dim the registers are laid out for, and with EXACT the head_dim itself (otherwise every step over
 * the dimensions asks whether it is needed, which keeps the compiler from overlapping them: 3 times the time of a
 * chunk at 128); CS: tokens of a chunk; NT: groups of eight query heads in a unit. */
template <class T, int DMAX, int CS, bool EXACT, int NT>
struct KvAttendWork {
    static constexpr int threads = 32 * (KV_WORKERS + 1), min_blocks = 2;
    static constexpr uint32_t smem = 112 * 1024;
    static constexpr uint32_t ring_bytes = (smem - 1024u - (uint32_t)sizeof(kv_shared_t)) & ~1023u;
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
    uint32_t ahead;                                      /* KV_AHEAD, or less in a small cache */
    uint32_t piece;                                      /* tokens of a chunk that are sure to lie in one page: CS or 16 */
    float scale_log2;                                    /* the scale's magnitude x log2(e); its sign goes into the query */
    uint32_t q_sign;
    uint32_t window, sinks;                              /* 0x7fffffff at most */
    uint32_t* arrived;                                   /* per worker, all ones at the start: arrivals at the unit it begins */
    float* parts;                                        /* [worker][2]: rows x head_dim sums, 16 maxima, 16 denominators */

    BAM_DEV uint32_t counters(uint32_t blocks) const { return blocks * KV_WORKERS; }
    BAM_DEV uint32_t dim() const { return EXACT ? (uint32_t)DMAX : L.head_dim; }
    BAM_DEV uint32_t row_bytes() const { return dim() * 2u; }
    BAM_DEV uint32_t stage_bytes() const { return CS * dim() * 4u; }
    BAM_DEV uint32_t stages() const
    {
        const uint32_t n = ring_bytes / (KV_WORKERS * stage_bytes());
        return n < KV_STAGES_MAX ? n : KV_STAGES_MAX;
    }
    BAM_DEV float* part(uint32_t worker, uint32_t which) const { return parts + ((size_t)worker * 2 + which) * (KV_ROWS * (dim() + 2)); }

    BAM_DEV kv_seen_t seen(uint32_t b, bool tell = false) const
    {
        kv_seen_t v;
        const int32_t len = __ldg(lens + b);
        v.len = (uint32_t)len;
        if (len < 0 || v.len > (uint64_t)table_width * L.block_tokens) {
            if (tell) L.bad_index((uint64_t)(int64_t)len);
            v.len = 0;
        }
        v.first = v.begin = v.len;
        if (window > 0 && window < v.len) {
            const uint32_t w0 = v.len - window;
            v.first = sinks < v.len ? sinks : v.len;
            if (w0 > v.first) v.begin = w0; else v.first = v.begin = v.len;
        }
        v.n_first = (v.first + CS - 1) / CS;
        v.from = v.begin / CS;
        if (v.from < v.n_first) v.from = v.n_first;
        const uint32_t end = (v.len + CS - 1) / CS;
        v.n = v.n_first + (end > v.from ? end - v.from : 0u);
        return v;
    }
    BAM_DEV static uint32_t first_token(const kv_seen_t& v, uint32_t c) { return (c < v.n_first ? c : v.from + (c - v.n_first)) * CS; }

    /* ---- the list ------------------------------------------------------------------------------------- */
    /* The list and the workers that share it: worker i takes the chunks from i * total / workers on (all differ by one
     * chunk at most).  Cuts that moved to the edge of a unit nearby saved joins and no time: 168 us both ways at 64
     * sequences of 2500-4100 tokens. */
    struct list_t {
        uint64_t total, workers;
        BAM_DEV uint64_t cut(uint64_t i) const { return i * total / workers; }
        BAM_DEV uint64_t worker_of(uint64_t x) const { return ((x + 1) * workers - 1) / total; }
    };

    /* Where worker i's run begins.  All lanes. */
    BAM_DEV kv_place_t begin_of(const kv_shared_t& sh, uint64_t i, const list_t& list) const
    {
        const uint32_t lane = lane_id(), units = L.n_kv_heads * tiles;
        kv_place_t p = { list.total, 0, 0 };
        if (i >= list.workers) return p;
        const uint64_t x = list.cut(i);
        uint32_t t = 0;
#pragma unroll
        for (uint32_t k = 0; k < KV_WORKERS + 1; k++) t += __popc(__ballot_sync(0xffffffffu, sh.before[k * 32 + lane] <= x));
        t -= 1;
        const uint32_t run = (batch + threads - 1) / threads;
        uint64_t at = sh.before[t];
        for (uint32_t b0 = t * run;; b0 += 32) {                    /* the sequence in the thread's run */
            const uint32_t b = b0 + lane;
            uint64_t span = b < batch && b < (t + 1) * run ? (uint64_t)seen(b).n * units : 0u, upto = span;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += y;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, x < at + upto);
            if (m == 0u) {
                at += __shfl_sync(0xffffffffu, upto, 31);
                if (b0 + 32 >= (t + 1) * run) return p;             /* the lengths changed under the launch */
                continue;
            }
            const uint32_t src = __ffs(m) - 1;
            p.b = b0 + src;
            at += __shfl_sync(0xffffffffu, upto - span, src);
            break;
        }
        p.f = x;
        p.pos = x - at;
        return p;
    }
    /* the first worker of the unit [U0, U1), and how many there are */
    BAM_DEV static void workers_of(uint64_t U0, uint64_t U1, const list_t& list, uint32_t& first, uint32_t& count)
    {
        const uint64_t i0 = list.worker_of(U0);
        first = (uint32_t)i0;
        count = (uint32_t)(list.worker_of(U1 - 1) - i0 + 1);
    }

    /* ---- pages and copies ----------------------------------------------------------------------------- */
    /* A warp's wait, and it ends: `done`, asked by all lanes together, says when; false when the block gives up
     * (someone's wait ran out, or the status block says so). */
    template <class Done>
    BAM_DEV bool wait(kv_shared_t& sh, Done done) const
    {
        uint32_t polls = 0;
        uint64_t t0 = 0;
        while (!done()) {
            bool stop = sh.abort;
            if (((++polls) & 255u) == 0u) {
                bam_status_t* st = L.r.cache.status;
                const uint64_t now = global_timer_ns();
                if (t0 == 0) t0 = now;
                /* the waits inside an acquire have one limit each; twice that is more than it needs to report */
                if (now - t0 > 2 * st->spin_timeout_ns) status_fail(st, BAM_ETIMEDOUT, BAM_AT_TMA, polls);
                stop |= status_bad(st);
            }
            if (__any_sync(0xffffffffu, stop)) { sh.abort = 1; return false; }
        }
        return true;
    }

    /* The pinning warp: KV_PIN_LANES lanes work for each worker, one page each. */
    BAM_DEV void pin_ahead(kv_shared_t& sh, uint32_t vb) const
    {
        const uint32_t full_mask = 0xffffffffu, lane = lane_id(), pieces = CS / piece, units = L.n_kv_heads * tiles;
        const bool works = lane < KV_WORKERS * KV_PIN_LANES;
        const uint32_t w = works ? lane / KV_PIN_LANES : 0, i = lane - w * KV_PIN_LANES, c = i / pieces, k = i - c * pieces;
        const uint32_t mask = ((1u << KV_PIN_LANES) - 1u) << (w * KV_PIN_LANES);       /* the lanes of my worker */
        const uint32_t most = KV_PIN_LANES / pieces < ahead ? KV_PIN_LANES / pieces : ahead;
        const uint32_t end = works ? sh.chunks[w] : 0;
        kv_place_t at = sh.from[w];                       /* where chunk `next` of the worker is */
        uint32_t next = 0, ask = most;                    /* chunks asked for at a time: fewer in a cache that is too full for all */
        bool alone = false;                               /* one worker's next chunk and nothing else: no chunk could be had whole */
        spin_t sp;
        for (;;) {
            const uint32_t n = next + c, round = n / ahead, place = n - round * ahead;
            bool mine = false;
            /* the next chunks that have a place */
            if (!wait(sh, [&] {
                    mine = n < end && c < ask && ld_acquire_cta(&sh.tag[w][place]) == 2u * round;
                    return __any_sync(full_mask, mine) || __all_sync(full_mask, next >= end);
                })) return;
            if (!__any_sync(full_mask, mine)) return;     /* all runs are pinned */
            const uint32_t gap = ~__ballot_sync(full_mask, mine) & mask;                 /* (the places come free in order) */
            if (gap && lane > (uint32_t)__ffs(gap) - 1u) mine = false;
            if (alone && ((__ballot_sync(full_mask, mine) & ((1u << lane) - 1u) & ~mask) || c > 0)) mine = false;
            uint32_t b = at.b, rows = 0, slot = BAM_SLOT_NONE;
            uint64_t pos = at.pos + c, page = 0, offset = 0;
            bool want = false;
            if (mine) {
                kv_seen_t v = seen(b);
                while (pos >= (uint64_t)v.n * units && b + 1 < batch) { pos -= (uint64_t)v.n * units; v = seen(++b); }
                if (pos >= (uint64_t)v.n * units) {                                      /* the lengths changed under the launch */
                    status_fail(L.r.cache.status, BAM_EINVAL, BAM_AT_RANGE, v.len);
                    sh.abort = 1;
                    v.n = 1;
                    pos = 0;
                }
                const uint32_t u = (uint32_t)(pos / v.n), ci = (uint32_t)(pos - (uint64_t)u * v.n);
                const uint32_t t0 = first_token(v, ci), tb = t0 + k * piece;
                uint32_t lo = tb, hi = tb + piece < v.len ? tb + piece : v.len;
                if (tb >= v.first && lo < v.begin) lo = v.begin;
                if (tb + piece <= v.begin && hi > v.first) hi = v.first;
                if (lo < hi) {
                    const int64_t block = __ldg(table + b * table_stride + tb / L.block_tokens);
                    if (block < 0 || (uint64_t)block >= L.n_blocks) L.bad_index((uint64_t)block);
                    else {
                        want = true;
                        page = L.page_of((uint64_t)block, u / tiles);
                        rows = (lo - t0) << 16 | (hi - lo);
                        offset = (uint64_t)(lo % L.block_tokens) * row_bytes();
                    }
                }
            }
            slot = kv_pin_warp(L, want, page, false, vb * KV_WORKERS);
            const bool got = want && slot <= BAM_SLOT_MAX;
            const bool failed = __any_sync(full_mask, want && slot == BAM_SLOT_ERR);
            /* What could not be had is asked for again; the chunks of the worker behind it give theirs back meanwhile, and
             * those before it are handed on.  So what a block holds pinned is always what its workers consume without
             * anybody's help, and blocks never wait for pages that wait for them. */
            const uint32_t miss = __ballot_sync(full_mask, want && !got) & mask, taken = __ballot_sync(full_mask, mine) & mask;
            const uint32_t ready = (miss ? __ffs(miss) - 1u - w * KV_PIN_LANES : (uint32_t)__popc(taken)) / pieces;     /* chunks */
            if (got && (c >= ready || failed)) L.r.release_page(slot, 1);
            if (failed) { sh.abort = 1; return; }
            if (mine && c < ready) {
                kv_pinned_t* e = &sh.pinned[w][place];
                e->src[k] = got ? L.r.get_cache_page_addr(slot) + offset : 0;
                e->slot[k] = got ? slot : BAM_SLOT_NONE;
                e->rows[k] = got ? rows : 0;
            }
            __syncwarp();
            if (mine && c < ready && k == 0) st_release_cta(&sh.tag[w][place], 2u * round + 1u);
            const uint32_t last = w * KV_PIN_LANES + (ready ? ready * pieces - 1 : 0);
            const uint32_t lb = __shfl_sync(full_mask, b, last);
            const uint64_t lpos = __shfl_sync(full_mask, pos, last);
            if (ready) { next += ready; at.b = lb; at.pos = lpos + 1; }
            ask = miss ? (ask + 1) / 2 : (ask * 2 < most ? ask * 2 : most);
            alone = !__any_sync(full_mask, ready);
            if (alone) {
                if (__any_sync(full_mask, sp.expired(L.r.cache.status, BAM_AT_FIND_SLOT, page))) { sh.abort = 1; return; }
            } else sp.reset();
        }
    }

    /* A worker's pipeline. */
    struct pipe_t {
        uint32_t base, w;               /* shared address of the worker's stages; its number in the block */
        uint32_t end;                   /* chunks of the run                                              */
        uint32_t next, stage, use;      /* the chunk that is consumed next, its stage and how often that was used before */
        uint32_t next_place, next_round;
        uint32_t issue, issue_stage;    /* the chunk that is copied next                                  */
        uint32_t issue_place, issue_round;
    };

    /* Start the copies of the worker's next chunk, if it has a free stage and the chunk is pinned; false if not. */
    BAM_DEV bool issue_next(kv_shared_t& sh, pipe_t& g) const
    {
        if (g.issue >= g.end || g.issue - g.next >= stages()) return false;
        const uint32_t lane = lane_id();
        if (!__all_sync(0xffffffffu, ld_acquire_cta(&sh.tag[g.w][g.issue_place]) == 2u * g.issue_round + 1u)) return false;
        if (lane == 0) {
            const kv_pinned_t e = sh.pinned[g.w][g.issue_place];
            const uint32_t full = smem_u32(&sh.full[g.w][g.issue_stage]), dst = g.base + g.issue_stage * stage_bytes();
            const uint32_t n0 = (e.rows[0] & 0xffffu) * row_bytes(), n1 = piece < CS ? (e.rows[1] & 0xffffu) * row_bytes() : 0;
            /* pages that this launch fetched were written by bulk copies too; order those before ours */
            asm volatile("fence.proxy.async.global;" ::: "memory");
            mbar_expect_tx(full, 2 * (n0 + n1));
            if (n0) {
                const uint32_t d = dst + (e.rows[0] >> 16) * row_bytes();
                bulk_load(d, reinterpret_cast<const void*>(e.src[0]), n0, full);
                bulk_load(d + CS * row_bytes(), reinterpret_cast<const void*>(e.src[0] + L.v_offset()), n0, full);
            }
            if (n1) {
                const uint32_t d = dst + (e.rows[1] >> 16) * row_bytes();
                bulk_load(d, reinterpret_cast<const void*>(e.src[1]), n1, full);
                bulk_load(d + CS * row_bytes(), reinterpret_cast<const void*>(e.src[1] + L.v_offset()), n1, full);
            }
        }
        __syncwarp();
        g.issue++;
        if (++g.issue_stage == stages()) g.issue_stage = 0;
        if (++g.issue_place == ahead) { g.issue_place = 0; g.issue_round++; }
        return true;
    }

    /* Wait until the next chunk has landed, and start copies of later ones meanwhile. */
    BAM_DEV bool landed(kv_shared_t& sh, pipe_t& g) const
    {
        const uint32_t full = smem_u32(&sh.full[g.w][g.stage]);
        return wait(sh, [&] {
            while (issue_next(sh, g)) {}
            return g.next < g.issue && __all_sync(0xffffffffu, mbar_test(full, g.use & 1u));
        });
    }
    /* The next chunk has landed: unpin its pages.  The rows are in shared memory, nothing of this thread is outstanding
     * that a release would have to wait for; its fence held the warp up for 2000 cycles a chunk. */
    BAM_DEV void unpin(kv_shared_t& sh, const pipe_t& g) const
    {
        const uint32_t lane = lane_id();
        if (lane < CS / piece) {
            const uint32_t slot = sh.pinned[g.w][g.next_place].slot[lane];
            if (slot != BAM_SLOT_NONE) red_add_relaxed(&L.r.cache.slots[slot].state, 0u - 1u);
        }
        __syncwarp();
        if (lane == 0) st_release_cta(&sh.tag[g.w][g.next_place], 2u * g.next_round + 2u);
    }
    BAM_DEV void advance(pipe_t& g) const
    {
        g.next++;
        if (++g.stage == stages()) { g.stage = 0; g.use++; }
        if (++g.next_place == ahead) { g.next_place = 0; g.next_round++; }
    }

    /* ---- products ------------------------------------------------------------------------------------- */
    /* the query fragments: rows lane / 4 and lane / 4 + 8 of the unit, head_dim in steps of 16 */
    BAM_DEV void load_q(uint32_t (&a)[DMAX / 16][4], const uint16_t* r0, const uint16_t* r1) const
    {
        const uint32_t d0 = (lane_id() & 3u) * 2;
        if (q32) {
#pragma unroll
            for (int i = 0; i < DMAX / 4; i++) {
                const uint16_t* r = i & 1 ? r1 : r0;
                const uint32_t d = (i >> 2) * 16 + d0 + (i & 2) * 4;
                a[i >> 2][i & 3] = r && (EXACT || (i >> 2) * 16 < (int)L.head_dim) ? __ldg(reinterpret_cast<const uint32_t*>(r + d)) : 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < DMAX / 4; i++) {
                const uint16_t* r = i & 1 ? r1 : r0;
                const uint32_t d = (i >> 2) * 16 + d0 + (i & 2) * 4;
                a[i >> 2][i & 3] = r && (EXACT || (i >> 2) * 16 < (int)L.head_dim) ? (uint32_t)__ldg(r + d) | ((uint32_t)__ldg(r + d + 1) << 16) : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < DMAX / 4; i++) a[i >> 2][i & 3] ^= q_sign;
    }

    /* The running softmax.  Thread (r, c) = (lane / 4, lane % 4) holds m and l of queries r and r + 8 (its share of l),
     * and of the sums the dimensions 16 i + r and + 8 of queries 8 n + 2 c and + 1. */
    struct state_t {
        float o[NT][DMAX / 16][4];
        float m[2], l[2];
    };
    /* a score's weight beside a maximum, both unscaled */
    BAM_DEV float weight_of(float s, float m) const { return exp2_fast((s - m) * scale_log2); }
    /* what a thread knows of queries lane / 4 and lane / 4 + 8, for the queries of its columns */
    BAM_DEV static void to_columns(float x0, float x1, float (&c)[NT][2])
    {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t src = ((lane_id() & 3u) * 2 + e) * 4;
            c[0][e] = __shfl_sync(0xffffffffu, x0, src);
            if (NT == 2) c[NT - 1][e] = __shfl_sync(0xffffffffu, x1, src);
        }
    }

    /* One chunk: S = Q K^T, p = 2^((S - m) scale log2(e)), O^T += V^T p^T.  m is a maximum of S as it is, and the difference
     * comes before the scale: the largest weight is 1 however large the scores are.  (With a scaled m it would be 2 to the
     * rounding of m, anything beyond 2^24.)  The weights go into the product as two 16-bit parts,
     * kv_type::weight p = hi + lo, which keeps 16 bits of them (bf16), or 21 and what is above 2^-40 (fp16): the product
     * runs twice, on a pipe that idles.  The sums are of the same scale, the denominator counts p itself.
     * An infinite value makes its sum infinite, if its weight is any number but 0 in 32 bits: infinity x 0, of a part that
     * is 0, and infinities of different sign, of parts of different sign, would make it NaN.  So hi is never 0 (lo takes what
     * is too much back) and lo is multiplied with values cut to the finite range.
     * There is one copy of this code, for whole chunks and others: code that runs once a unit runs from a cold
     * instruction cache, at a microsecond for every few kilobytes. */
    BAM_DEV void chunk(state_t& z, const uint32_t (&qa)[DMAX / 16][4], uint32_t stage, const kv_seen_t& v, uint32_t t0) const
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
        if (!(t0 + CS <= v.first || (t0 >= v.begin && t0 + CS <= v.len))) {
            /* rows that are not visible may hold anything.  Their scores become -infinity and their values zeros: their
             * weights are 0, and 0 x NaN is not 0 */
#pragma unroll
            for (int i = 0; i < CS / 4; i++) {
                const uint32_t j = t0 + (i >> 1) * 8 + (lane & 3u) * 2 + (i & 1);
                if (!((j < v.first || j >= v.begin) && j < v.len)) s[i >> 1][i & 1] = s[i >> 1][2 + (i & 1)] = -INFINITY;
            }
#pragma unroll 1
            for (uint32_t i = lane; i < CS * (dim() / 8); i += 32) {
                const uint32_t j = t0 + i / (dim() / 8);
                if (!((j < v.first || j >= v.begin) && j < v.len))
                    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(stage + CS * rb + i * 16u), "r"(0u) : "memory");
            }
            /* the stage's next rows come through the other proxy */
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < CS / 8; i++) {
            mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][1]));
            mx1 = fmaxf(mx1, fmaxf(s[i][2], s[i][3]));
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float n0 = fmaxf(z.m[0], mx0), n1 = fmaxf(z.m[1], mx1);
        const float c0 = n0 == -INFINITY ? 0.f : n0, c1 = n1 == -INFINITY ? 0.f : n1;     /* nothing seen yet: exp2(-inf - 0) = 0 */
        if (__any_sync(0xffffffffu, n0 != z.m[0] || n1 != z.m[1])) {
            const float a0 = weight_of(z.m[0], c0), a1 = weight_of(z.m[1], c1);
            float a[NT][2];
            to_columns(a0, a1, a);
            z.l[0] *= a0; z.l[1] *= a1;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < DMAX / 16; i++) { z.o[n][i][0] *= a[n][0]; z.o[n][i][1] *= a[n][1]; z.o[n][i][2] *= a[n][0]; z.o[n][i][3] *= a[n][1]; }
            z.m[0] = n0; z.m[1] = n1;
        }
        const uint32_t v_row = stage + CS * rb + ((lane & 7u) + ((lane >> 4) & 1u) * 8u) * rb, v_c = (lane >> 3) & 1u;
        uint32_t hi[NT][CS / 8], lo[NT][CS / 8];
#pragma unroll
        for (int i = 0; i < CS / 8; i++) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float p[2];
#pragma unroll
                for (int e = 0; e < 2; e++) p[e] = weight_of(s[i][2 * n + e], n ? c1 : c0);
                z.l[n] += p[0] + p[1];
                const float w0 = p[0] * kv_type<T>::weight, w1 = p[1] * kv_type<T>::weight;
                hi[n][i] = kv_type<T>::positive(kv_type<T>::pack(w0, w1));
                const float2 h = kv_type<T>::unpack(hi[n][i]);
                lo[n][i] = kv_type<T>::pack(w0 - h.x, w1 - h.y);
            }
        }
#pragma unroll
        for (int kt = 0; kt < CS / 16; kt++) {
#pragma unroll
            for (int mt = 0; mt < DMAX / 16; mt++) {
                if (EXACT || mt * 16 < (int)L.head_dim) {
                    uint32_t r[4];
                    ldm_x4_t(r, at(v_row, v_c, mt * 2) + kt * 16 * rb);
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_16816(z.o[n][mt], r, hi[n][2 * kt], hi[n][2 * kt + 1], T());
#pragma unroll
                    for (int k = 0; k < 4; k++) r[k] = kv_type<T>::finite(r[k]);
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_16816(z.o[n][mt], r, lo[n][2 * kt], lo[n][2 * kt + 1], T());
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
    /* what the sums are multiplied with in the end */
    BAM_DEV static float inverse(float l) { return l == 0.f ? 0.f : (1.f / kv_type<T>::weight) / l; }
    /* nothing visible: -infinity twice over; scores that are all NaN leave m at -infinity, and l says NaN */
    BAM_DEV float lse_of(float m, float l) const { return m * scale_log2 * 0.69314718055994531f + logf(l); }

    /* the unit's result from one warp's registers */
    BAM_DEV void write_out(const state_t& z, uint32_t b, uint32_t u) const
    {
        const uint32_t lane = lane_id(), h = u / tiles, r0 = (u - h * tiles) * KV_ROWS;
        float inv[NT][2];
        to_columns(inverse(z.l[0]), inverse(z.l[1]), inv);
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t r = r0 + 8 * n + (lane & 3u) * 2 + e;
                uint16_t* p = out + b * o_sb + (h * group + r) * o_sh;
#pragma unroll
                for (int i = 0; i < DMAX / 16; i++) {
                    if (EXACT || i * 16 < (int)L.head_dim) {
                        /* neighbours in a row of the output sit four lanes apart: the even row of threads takes a pair from
                         * the dimensions r, the odd one from r + 8 */
                        const float a = z.o[n][i][e] * inv[n][e], c = z.o[n][i][2 + e] * inv[n][e];
                        const bool odd = lane & 4u;
                        const float other = __shfl_xor_sync(0xffffffffu, odd ? a : c, 4);
                        if (r < group) store_pair(p + i * 16 + (odd ? 8 : 0) + ((lane >> 2) & 6u), odd ? other : a, odd ? c : other);
                    }
                }
            }
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = r0 + (lane >> 2) + 8 * half;
            if (lse && (lane & 3u) == 0u && r < group) lse[(size_t)b * n_q_heads + h * group + r] = lse_of(z.m[half], z.l[half]);
        }
    }
    /* query heads of unit u */
    BAM_DEV uint32_t rows_of(uint32_t u) const
    {
        const uint32_t r0 = u % tiles * KV_ROWS;
        return group - r0 < KV_ROWS ? group - r0 : KV_ROWS;
    }
    /* A part of a unit in the scratch: maxima and denominators by query, and the sums as the registers hold them, quad
     * [n][i][lane]: dimensions 16 i + lane / 4 and + 8 of queries 8 n + 2 (lane % 4) and + 1. */
    BAM_DEV void write_part(const state_t& z, float* p, uint32_t rows) const
    {
        const uint32_t lane = lane_id();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < DMAX / 16; i++)
                if ((EXACT || i * 16 < (int)L.head_dim) && 8 * n + (lane & 3u) * 2 < rows) {
                    float* q_ = p + ((n * (dim() / 16) + i) * 32 + lane) * 4;
                    st_cg_f4(q_, z.o[n][i][0], z.o[n][i][1], z.o[n][i][2], z.o[n][i][3]);
                }
        if ((lane & 3u) == 0u) {
            float* ml = p + KV_ROWS * dim() + 2 * (lane >> 2);
            st_cg_f2(ml, z.m[0], z.l[0]);
            st_cg_f2(ml + 16, z.m[1], z.l[1]);
        }
    }

    /* ---- a worker ------------------------------------------------------------------------------------- */
    BAM_DEV void work(kv_shared_t& sh, uint32_t ring, const list_t& list, uint32_t worker) const
    {
        const uint32_t lane = lane_id(), w = threadIdx.x >> 5, units = L.n_kv_heads * tiles;
        pipe_t g;
        g.base = ring + w * stages() * stage_bytes(); g.w = w;
        const kv_place_t from = sh.from[w];
        g.end = sh.chunks[w];
        g.next = g.stage = g.use = g.issue = g.issue_stage = g.next_place = g.next_round = g.issue_place = g.issue_round = 0;
        const uint64_t f1 = from.f + g.end;
        uint32_t b = from.b, n_join = 0;
        uint64_t pos = from.pos;
        for (uint64_t f = from.f; f < f1;) {
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
            for (int i = 0; i < NT * (DMAX / 16); i++) { float* o = z.o[i / (DMAX / 16)][i % (DMAX / 16)]; o[0] = o[1] = o[2] = o[3] = 0.f; }
            z.m[0] = z.m[1] = -INFINITY;
            z.l[0] = z.l[1] = 0.f;
            uint32_t qa[DMAX / 16][4];
            load_q(qa, q0, q1);
            for (uint32_t i = 0; i < seg; i++) {
                if (!landed(sh, g)) break;
                unpin(sh, g);
                const uint32_t stage = g.base + g.stage * stage_bytes();
                chunk(z, qa, stage, v, first_token(v, c + i));
                __syncwarp();
                advance(g);
            }
            if (__any_sync(0xffffffffu, sh.abort)) break;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                z.l[half] += __shfl_xor_sync(0xffffffffu, z.l[half], 1);
                z.l[half] += __shfl_xor_sync(0xffffffffu, z.l[half], 2);
            }
            if (seg == v.n) write_out(z, b, u);
            else {
                const uint64_t U0 = f - c;
                uint32_t i0, cnt;
                workers_of(U0, U0 + v.n, list, i0, cnt);
                write_part(z, part(worker, worker == i0 ? 1 : 0), rows_of(u));
                __syncwarp();
                if (lane == 0) {
                    /* one release for the warp: what its other lanes wrote comes before it by the barrier */
                    red_add_release(arrived + i0, 1u);
                    sh.join[w][n_join].b = b; sh.join[w][n_join].u = u; sh.join[w][n_join].first = i0; sh.join[w][n_join].workers = cnt;
                }
                n_join++;
            }
            f += seg;
            pos += seg;
        }
        if (g.next < g.end) {
            /* given up: copies that are still under way land (bounded) before the block leaves */
            while (g.next < g.issue) {
                const uint64_t since = global_timer_ns();
                const uint32_t full = smem_u32(&sh.full[w][g.stage]);
                while (!mbar_test(full, g.use & 1u) && global_timer_ns() - since < 2 * L.r.cache.status->spin_timeout_ns) {}
                __syncwarp();
                unpin(sh, g);
                advance(g);
            }
            return;
        }
        __syncwarp();
        for (uint32_t k = 0; k < n_join; k++) join(sh.join[w][k].b, sh.join[w][k].u, sh.join[w][k].first, sh.join[w][k].workers, worker);
    }

    /* This worker's share of a unit that several worked on. */
    BAM_DEV void join(uint32_t b, uint32_t u, uint32_t i0, uint32_t cnt, uint32_t worker) const
    {
        const uint32_t lane = lane_id(), D = dim();
        bam_status_t* st = L.r.cache.status;
        uint32_t polls = 0, gone = 0;
        uint64_t t0 = 0;
        /* a warp whose pages are all in the cache may be done long before one whose pages come from the store: the limit is
         * that of the launch */
        if (lane == 0) {
            while (ld_acquire_gpu(arrived + i0) != cnt - 1u && !gone) {
                if (((++polls) & 63u) == 0u) {
                    const uint64_t now = global_timer_ns();
                    if (t0 == 0) t0 = now;
                    if (now - t0 > st->launch_timeout_ns) status_fail(st, BAM_ETIMEDOUT, BAM_AT_KV_JOIN, i0);
                    gone = status_bad(st) ? 1u : 0u;
                }
            }
        }
        if (__shfl_sync(0xffffffffu, gone, 0)) return;
        const uint32_t h = u / tiles, r0 = (u - h * tiles) * KV_ROWS;
        const uint32_t rows = rows_of(u), quads = (rows + 7) / 8 * (D / 16) * 32, j = worker - i0;
        const uint32_t g0 = quads * j / cnt, g1 = quads * (j + 1) / cnt;
        /* A quad is four elements of the output (see write_part); P lanes share one, each adds up to four parts of two quads
         * at a time, whose loads are all issued before the first is used: a part is one access to L2, and one after the
         * other they took 10 to 15 us of a call. */
        uint32_t P = 1;
        while (P * 4 < cnt && P < 32u) P <<= 1;
        const uint32_t p = lane & (P - 1u), at_once = 32u / P;
#pragma unroll 1
        for (uint32_t base = g0; base < g1; base += 2 * at_once) {
            /* of two queries, q0 and q0 + 1 */
            uint32_t gi[2], q0[2];
            bool act[2];
            float M[2][2], l[2][2], x[2][4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                gi[e] = base + e * at_once + lane / P;
                q0[e] = gi[e] / (32u * (D / 16)) * 8 + (gi[e] & 3u) * 2;
                act[e] = gi[e] < g1 && q0[e] < rows;
                M[e][0] = M[e][1] = -INFINITY;
                l[e][0] = l[e][1] = x[e][0] = x[e][1] = x[e][2] = x[e][3] = 0.f;
            }
#pragma unroll 1
            for (uint32_t s0 = 0; s0 < cnt; s0 += 4 * P) {
                uint4 ml[2][4], y[2][4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t s = s0 + k * P + p;
                    const float* y_ = part(i0 + s, s == 0 ? 1 : 0);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        ml[e][k] = make_uint4(0xff800000u, 0u, 0xff800000u, 0u);              /* -infinity, 0 */
                        y[e][k] = make_uint4(0, 0, 0, 0);
                        if (s < cnt && act[e]) {
                            ml[e][k] = ld_cg_v4(y_ + KV_ROWS * D + 2 * q0[e]);
                            y[e][k] = ld_cg_v4(y_ + (size_t)gi[e] * 4);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int c2 = 0; c2 < 2; c2++) {
                        float m = M[e][c2];
#pragma unroll
                        for (int k = 0; k < 4; k++) m = fmaxf(m, __uint_as_float(c2 ? ml[e][k].z : ml[e][k].x));
                        const float c = m == -INFINITY ? 0.f : m, a = weight_of(M[e][c2], c);
                        M[e][c2] = m;
                        l[e][c2] *= a; x[e][c2] *= a; x[e][2 + c2] *= a;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float a1 = weight_of(__uint_as_float(c2 ? ml[e][k].z : ml[e][k].x), c);
                            l[e][c2] += __uint_as_float(c2 ? ml[e][k].w : ml[e][k].y) * a1;
                            x[e][c2] += __uint_as_float(c2 ? y[e][k].y : y[e][k].x) * a1;
                            x[e][2 + c2] += __uint_as_float(c2 ? y[e][k].w : y[e][k].z) * a1;
                        }
                    }
                }
            }
            float all[2][2] = { { M[0][0], M[0][1] }, { M[1][0], M[1][1] } };
#pragma unroll 1
            for (uint32_t o = P >> 1; o > 0; o >>= 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) all[i >> 1][i & 1] = fmaxf(all[i >> 1][i & 1], __shfl_xor_sync(0xffffffffu, all[i >> 1][i & 1], o));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float a = weight_of(M[i >> 1][i & 1], all[i >> 1][i & 1] == -INFINITY ? 0.f : all[i >> 1][i & 1]);
                l[i >> 1][i & 1] *= a; x[i >> 1][i & 1] *= a; x[i >> 1][2 + (i & 1)] *= a;
            }
#pragma unroll 1
            for (uint32_t o = P >> 1; o > 0; o >>= 1) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) x[e][i] += __shfl_xor_sync(0xffffffffu, x[e][i], o);
                    l[e][0] += __shfl_xor_sync(0xffffffffu, l[e][0], o);
                    l[e][1] += __shfl_xor_sync(0xffffffffu, l[e][1], o);
                }
            }
            if (p == 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = i >> 1, c2 = i & 1;
                    if (act[e] && q0[e] + c2 < rows) {
                        const uint32_t hq = h * group + r0 + q0[e] + c2, d = gi[e] / 32 % (D / 16) * 16 + (gi[e] >> 2) % 8;
                        const float inv = inverse(l[e][c2]);
                        uint16_t* dst = out + b * o_sb + hq * o_sh + d;
                        const uint32_t w = kv_type<T>::pack(x[e][c2] * inv, x[e][2 + c2] * inv);
                        dst[0] = (uint16_t)w;
                        dst[8] = (uint16_t)(w >> 16);
                        if (lse && d == 0) lse[(size_t)b * n_q_heads + hq] = lse_of(all[e][c2], l[e][c2]);
                    }
                }
            }
        }
    }

    __device__ void operator()(uint32_t vb, uint32_t nvb) const
    {
        /* stages on 1 KB boundaries: the addresses within one are formed with XOR */
        uint8_t* const mem = bam_dyn_smem + (0u - smem_u32(bam_dyn_smem)) % 1024u;
        kv_shared_t& sh = *reinterpret_cast<kv_shared_t*>(mem + ring_bytes);
        const uint32_t ring = smem_u32(mem), t = threadIdx.x, lane = t & 31u, w = t >> 5;
        const uint32_t units = L.n_kv_heads * tiles;
        if (t < KV_WORKERS * KV_STAGES_MAX) mbar_init(smem_u32(&sh.full[0][t]), 1);
        if (t < KV_WORKERS * KV_AHEAD) sh.tag[0][t] = 0;
        if (t == 0) sh.abort = status_bad(L.r.cache.status) ? 1u : 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        /* how many chunks there are before each sequence: every thread counts a run of sequences */
        const uint32_t run = (batch + threads - 1) / threads;
        const uint32_t s0 = t * run < batch ? t * run : batch, s1 = s0 + run < batch ? s0 + run : batch;
        uint64_t own = 0;
        uint32_t longest = 0;
        for (uint32_t b = s0; b < s1; b++) {
            const uint32_t n = seen(b, vb == 0).n;
            own += n;
            longest = n > longest ? n : longest;
        }
        uint64_t before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= (uint32_t)o) before += x;
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        if (lane == 31) { sh.warp_sum[w] = before; sh.warp_max[w] = longest; }
        before -= own;
        __syncthreads();
        if (sh.abort) return;
        uint64_t total = 0;
#pragma unroll
        for (uint32_t k = 0; k < KV_WORKERS + 1; k++) {
            if (k < w) before += sh.warp_sum[k];
            total += sh.warp_sum[k];
            longest = sh.warp_max[k] > longest ? sh.warp_max[k] : longest;
        }
        total *= units;
        sh.before[t] = before * units;
        /* workers: all there are, but none of them with less than KV_MIN_CHUNKS (or the longest unit, if that is shorter) */
        const uint64_t n_workers = (uint64_t)nvb * KV_WORKERS, least = longest < KV_MIN_CHUNKS ? longest : KV_MIN_CHUNKS;
        list_t list = { total, total >= n_workers * least ? n_workers : total / (least ? least : 1u) };
        if (list.workers == 0) list.workers = 1;
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
        /* neighbours in the list on different SMs: the workers of a short list spread out */
        const uint32_t worker = w * nvb + vb;
        if (w < KV_WORKERS) {
            const kv_place_t from = begin_of(sh, worker, list);
            if (lane == 0) { sh.from[w] = from; sh.chunks[w] = from.f < total ? (uint32_t)(list.cut(worker + 1ull) - from.f) : 0u; }
        }
        __syncthreads();
        if (w < KV_WORKERS) {
            if (sh.chunks[w]) work(sh, ring, list, worker);
        } else pin_ahead(sh, vb);
        __syncthreads();
        if (sh.abort && t < KV_WORKERS * KV_AHEAD && (sh.tag[0][t] & 1u)) {            /* given up: what was pinned and never copied */
            const kv_pinned_t& e = sh.pinned[0][t];
            for (uint32_t k = 0; k < CS / piece; k++) if (e.slot[k] != BAM_SLOT_NONE) L.r.release_page(e.slot[k], 1);
        }
    }
};

template <class T, int DMAX, int CS, bool EXACT, int NT>
static int launch_attend_nt(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    typedef KvAttendWork<T, DMAX, CS, EXACT, NT> Work;
    Work w;
    memset(&w, 0, sizeof w);
    w.L = L;
    w.q = (const uint16_t*)p->q; w.out = (uint16_t*)p->out; w.lse = p->lse;
    w.q_sb = p->q_stride[0]; w.q_sh = p->q_stride[1]; w.o_sb = p->out_stride[0]; w.o_sh = p->out_stride[1];
    w.table = p->block_table; w.table_stride = p->table_stride; w.table_width = p->table_width; w.lens = p->seq_lens;
    w.batch = p->batch; w.n_q_heads = p->n_q_heads;
    w.group = p->n_q_heads / L.n_kv_heads; w.tiles = (w.group + KV_ROWS - 1) / KV_ROWS;
    /* neither 0 nor infinite: -infinity x 0, of a score that is not visible, and 0 x infinity, of the largest, would be NaN */
    w.scale_log2 = fminf(fmaxf(fabsf(p->scale) * 1.4426950408889634f, FLT_TRUE_MIN), FLT_MAX);
    w.q_sign = p->scale < 0.f ? 0x80008000u : 0u;
    w.window = p->window < 0x7fffffff ? (uint32_t)p->window : 0x7fffffffu;
    w.sinks = p->sinks < 0x7fffffff ? (uint32_t)p->sinks : 0x7fffffffu;
    w.q32 = ((uintptr_t)p->q & 3) == 0 && p->q_stride[0] % 2 == 0 && p->q_stride[1] % 2 == 0;
    w.o32 = ((uintptr_t)p->out & 3) == 0 && p->out_stride[0] % 2 == 0 && p->out_stride[1] % 2 == 0;
    uint8_t* base = (uint8_t*)scratch;
    const uint32_t most = kv_most_blocks(a);
    w.arrived = (uint32_t*)(base + sizeof(kv_launch_words_t));
    w.parts = (float*)(base + kv_parts_at(most * KV_WORKERS));
    w.piece = L.block_tokens % CS == 0 ? CS : 16;
    if (a->pc->d.n_slots < CS / w.piece) return BAM_EINVAL;                               /* a chunk's pages are pinned together */
    /* no more blocks than the longest sequences could keep busy */
    uint64_t chunks = ((uint64_t)p->table_width * L.block_tokens + CS - 1) / CS;
    if (chunks > 0x80000000u / CS) chunks = 0x80000000u / CS;                             /* lengths are 32-bit numbers */
    if (p->window > 0) {
        const uint64_t seen = (uint64_t)p->window / CS + (uint64_t)(p->sinks < (1ll << 40) ? p->sinks : (1ll << 40)) / CS + 4;
        if (seen < chunks) chunks = seen;
    }
    const uint32_t least = chunks < KV_MIN_CHUNKS ? (uint32_t)chunks : KV_MIN_CHUNKS;
    const uint64_t workers = (chunks * p->batch * L.n_kv_heads * w.tiles + least - 1) / least;
    const uint64_t want = (workers + KV_WORKERS - 1) / KV_WORKERS;
    const uint64_t blocks = want < most ? want : most;
    /* no more pinned than the cache has slots; two chunks all the same, or copies would not overlap (a cache that is too
     * full for that makes the pinning warps ask for less) */
    const uint64_t share = a->pc->d.n_slots / (blocks * KV_WORKERS * (CS / w.piece));
    w.ahead = share < 2 ? 2u : share < KV_AHEAD ? (uint32_t)share : KV_AHEAD;
    return kv_launch(a->pc->ctrl, w, blocks, scratch, (cudaStream_t)stream);
}

template <class T, int DMAX, int CS, bool EXACT>
static int launch_attend_as(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    return p->n_q_heads / L.n_kv_heads <= 8 ? launch_attend_nt<T, DMAX, CS, EXACT, 1>(a, L, p, scratch, stream)
                                            : launch_attend_nt<T, DMAX, CS, EXACT, 2>(a, L, p, scratch, stream);
}

template <class T>
int kv_launch_attend(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream)
{
    /* chunks of 32 tokens halve what a chunk costs beside its products (softmax statistics, barriers); above 128
     * dimensions their sums and scores do not fit the registers */
    switch (L.head_dim) {
    case 64: return launch_attend_as<T, 64, 32, true>(a, L, p, scratch, stream);
    case 80: return launch_attend_as<T, 80, 32, true>(a, L, p, scratch, stream);
    case 96: return launch_attend_as<T, 96, 32, true>(a, L, p, scratch, stream);
    case 128: return launch_attend_as<T, 128, 32, true>(a, L, p, scratch, stream);
    case 256: return launch_attend_as<T, 256, 16, true>(a, L, p, scratch, stream);
    default: break;
    }
    if (L.head_dim < 128) return launch_attend_as<T, 128, 16, false>(a, L, p, scratch, stream);
    return launch_attend_as<T, 256, 16, false>(a, L, p, scratch, stream);
}

}  // namespace bam
#endif
