/*
 * bam_kv.cuh -- rows of a key/value cache inside the pages of an array.
 *
 * A page of the array holds the keys and then the values of one block of `block_tokens` consecutive tokens for
 * ONE key/value head: page = first_page + block * n_kv_heads + head, and inside it
 *
 *     K[block_tokens][head_dim]  V[block_tokens][head_dim]          (16-bit elements)
 *
 * so that what one head needs of a block is one contiguous piece: one look-up, one pin, two bulk copies.
 * The 16-byte chunks of a row are permuted by the row's number (swizzle, below): eight consecutive rows then put
 * the same logical chunk on eight different 16-byte bank groups of shared memory, and the matrix loads of the
 * attention kernel read a page's verbatim copy without bank conflicts -- nobody has to permute on the way in.
 */
#ifndef BAM_KV_CUH
#define BAM_KV_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bam_abi.h"
#include "bam_fused.cuh"

namespace bam {

#define KV_ROWS 16u                   /* query heads of a unit of the attention: the rows of a matrix instruction */
#define KV_WORKERS 3u                 /* worker warps of a block of the attention; with the fourth, which only a controller
                                       * block uses, a thread may have 255 registers */

/* A launch's own words at the head of its scratch.  They (and the counters behind them) are all ones when a launch starts,
 * and the last of its blocks leaves them so for the next one that uses the scratch: no memset per launch.
 *   remaining  what the controller blocks watch; the last worker block clears it
 *   left       counts down.  Bits 0-14: worker blocks; bit 15: cleared when an index was outside its range; bits 16-31: all
 *              blocks.  (An index outside its range is noted in bad_index and goes into the status block by the last worker
 *              block: a status that is set earlier makes every wait of the launch give up, and a page whose fetch is given
 *              up is lost to the cache.)
 *   drawn      items that were drawn */
struct kv_launch_words_t {
    uint32_t remaining, left;
    uint64_t bad_index;
    uint32_t drawn, pad[11];
};

/* what a kernel knows of the layout */
struct kv_layout_d_t {
    range_d_t<uint64_t> r;
    uint64_t first_page, n_blocks;
    uint32_t head_dim, n_kv_heads, block_tokens;
    uint32_t chunks;                 /* 16-byte chunks of a row: head_dim / 8                 */
    uint32_t swz_shift, swz_mask;    /* see swizzle                                           */
    kv_launch_words_t* words;

    BAM_DEV void bad_index(uint64_t i) const
    {
        st_relaxed_gpu(&words->bad_index, i);
        (void)atom_and_release(&words->left, ~0x8000u);
    }
    /* the number of draws before this one; a warp draws together */
    BAM_DEV uint32_t draw() const
    {
        uint32_t n = 0;
        if (lane_id() == 0) n = atom_add_relaxed(&words->drawn, 1u) + 1u;
        return __shfl_sync(0xffffffffu, n, 0);
    }
    BAM_DEV uint64_t page_of(uint64_t block, uint32_t head) const { return first_page + block * n_kv_heads + head; }
    BAM_DEV uint32_t row_bytes() const { return head_dim * 2u; }
    BAM_DEV uint32_t v_offset() const { return block_tokens * head_dim * 2u; }
    /* Rows lie head_dim / 8 chunks apart.  With a multiple of 8 every row starts on the same bank group, so the
     * chunk number is XORed with the row's low three bits; with 4 mod 8 two rows make one round of the bank groups
     * and bits 2:1 of the row suffice, with 2 mod 4 bit 2.  An odd number needs none.  The mask's range divides
     * the number of chunks, so the result is a chunk of the same row. */
    BAM_DEV uint32_t swizzle(uint32_t row, uint32_t chunk) const { return chunk ^ ((row >> swz_shift) & swz_mask); }
};

/* weight: what the softmax weights, 1 at most, are multiplied with for the product with the values.  fp16 has no number
 * between 0 and 2^-24, but thousands of weights of that size beside one of 1 are a part of the output that it can tell from
 * none; 2^15 is the largest power of two below its maximum.  bf16 has the range of 32 bits.
 * positive: both elements of a weight (none is negative), none of them 0 for a weight that is not; in bf16 none is.
 * finite: both elements, an infinite one as the largest number of its sign. */
template <class T> struct kv_type;
template <> struct kv_type<__nv_bfloat16> {
    static constexpr float weight = 1.f;
    static BAM_DEV uint32_t positive(uint32_t u) { return u; }
    static BAM_DEV uint32_t finite(uint32_t u) { uint32_t r; asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x7f7f7f7fu)); return r; }
    static BAM_DEV uint32_t pack(float lo, float hi) { __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&p); }
    static BAM_DEV float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
};
template <> struct kv_type<__half> {
    static constexpr float weight = 32768.f;
    static BAM_DEV uint32_t positive(uint32_t u) { uint32_t r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x00010001u)); return r; }
    static BAM_DEV uint32_t finite(uint32_t u) { uint32_t r; asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x7bff7bffu)); return r; }
    static BAM_DEV uint32_t pack(float lo, float hi) { __half2 p = __floats2half2_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&p); }
    static BAM_DEV float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
};

/* Pin a page per lane: every lane calls it, lanes that want the same page share one fetch-add (each releases its own
 * count of one).  What is resident is pinned at once; the warp asks the cache's miss path for the rest. */
BAM_DEV uint32_t kv_pin_warp(const kv_layout_d_t& L, bool want, uint64_t page, bool write, uint32_t queue)
{
    const uint32_t full = 0xffffffffu, lane = lane_id();
    const uint32_t eq = __match_any_sync(full, want ? page : ~(uint64_t)lane);
    const uint32_t leader = __ffs(eq) - 1, cnt = __popc(eq);
    const bool ask = want && lane == leader;
    uint32_t slot = BAM_SLOT_ERR;
    if (ask) slot = cache_try_pin(L.r.cache, L.r.get_global_address(page), cnt, write);
    const uint32_t hits = __reduce_add_sync(full, ask && slot <= BAM_SLOT_MAX ? cnt : 0u);
    if (hits && lane == 0) count_hit(L.r.cache, hits);
    const bool more = ask && slot == BAM_SLOT_NONE;
    if (__any_sync(full, more)) {
        const uint32_t x = L.r.acquire_page_warp(full, more, more ? page : 0, cnt, write, queue);
        if (more) slot = x;
    }
    return __shfl_sync(full, slot, leader);
}

/* Eight elements from memory of any 2-byte alignment; `vec`: 16-byte aligned. */
BAM_DEV uint4 kv_load8(const uint16_t* p, bool vec)
{
    if (vec) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
BAM_DEV void kv_store8(uint16_t* p, uint4 v, bool vec)
{
    if (vec) { *reinterpret_cast<uint4*>(p) = v; return; }
    const uint32_t w[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
    for (int i = 0; i < 4; i++) { p[2 * i] = (uint16_t)w[i]; p[2 * i + 1] = (uint16_t)(w[i] >> 16); }
}

/* The fused launch of these operators.  Like bam_fused, but the words that end the controller blocks belong to the launch
 * and not to the controller, so that launches on one controller may overlap and a captured launch can be replayed.
 * Work::counters() of the words behind the launch's own are the workload's. */
template <class Work>
__global__ void __launch_bounds__(Work::threads, Work::min_blocks)
bam_kv_fused(const __grid_constant__ bam_emu_d_t emu, const __grid_constant__ Work work)
{
    kv_launch_words_t* const words = reinterpret_cast<kv_launch_words_t*>(emu.consumers_remaining);
    const bool controls = blockIdx.x < emu.n_ctrl_blocks;
    const uint32_t n_work = gridDim.x - emu.n_ctrl_blocks;
    if (controls) emu_controller_main(emu, bam_dyn_smem);
    else work(blockIdx.x - emu.n_ctrl_blocks, n_work);
    __syncthreads();
    /* (in the dynamic shared memory, which nobody uses any more: 128 bytes of their own would take three blocks of the gather
     * over 196 KB an SM, and half of the L1 with it: 55 -> 60 us) */
    uint32_t* const old_left = reinterpret_cast<uint32_t*>(bam_dyn_smem);
    if (threadIdx.x == 0) {
        /* nothing is published here: what the launch wrote becomes visible with its end */
        const uint32_t old = atom_add_relaxed(&words->left, controls ? 0u - 0x10000u : 0u - 0x10001u);
        if (!controls && (old & 0x7fffu) == 0x8000u - n_work) {                       /* the last of the workers */
            if (!(old & 0x8000u)) {
                fence_acq_rel_gpu();
                status_fail(emu.status, BAM_ERANGE, BAM_AT_RANGE, ld_relaxed_gpu(&words->bad_index));
            }
            st_release_scoped(&words->remaining, 0u, emu.sys_scope != 0);
        }
        *old_left = old;
    }
    __syncthreads();
    if ((*old_left >> 16) != 0x10000u - gridDim.x) return;
    /* the last block of all: nobody reads or writes the words any more (whether the launch succeeded or was given up) */
    uint32_t* w = reinterpret_cast<uint32_t*>(words);
    for (uint32_t i = threadIdx.x; i < sizeof(kv_launch_words_t) / 4 + work.counters(n_work); i += blockDim.x) w[i] = 0xffffffffu;
}

/* ---- host side ------------------------------------------------------------------------------------------ */


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

/* Launch with at most `want` worker blocks.  The launch's words are the first bytes of `scratch`. */
template <class Work>
int kv_launch(bam_ctrl* c, const Work& work, uint64_t want, void* scratch, cudaStream_t s)
{
    uint32_t grid = 0;
    CK(kv_max_grid<Work>(c->device, &grid));
    if (c->max_grid && grid > c->max_grid) grid = c->max_grid;
    bam_emu_d_t emu = c->emu;
    if (want == 0) want = 1;
    /* few workers need few command processors, but one for each queue: a processor that polls several of them in turn
     * sees the end of the launch a round trip later for each */
    const uint64_t few = want > (emu.n_qps + BAM_EMU_WARPS - 1) / BAM_EMU_WARPS ? want : (emu.n_qps + BAM_EMU_WARPS - 1) / BAM_EMU_WARPS;
    if (emu.n_ctrl_blocks > few) emu.n_ctrl_blocks = (uint32_t)few;
    if (grid <= emu.n_ctrl_blocks) return BAM_EINVAL;
    if (grid - emu.n_ctrl_blocks > want) grid = emu.n_ctrl_blocks + (uint32_t)want;
    emu.consumers_remaining = reinterpret_cast<uint32_t*>(scratch);
    Work w = work;
    w.L.words = reinterpret_cast<kv_launch_words_t*>(scratch);
    void* args[] = { (void*)&emu, (void*)&w };
    CK(cudaLaunchCooperativeKernel((const void*)bam_kv_fused<Work>, dim3(grid), dim3(Work::threads), args, Work::smem, s));
    return BAM_OK;
}

/* Scratch: the launch's words, a counter per worker warp of the attention, the workers' parts. */
inline uint32_t kv_most_blocks(bam_array* a) { return (uint32_t)a->pc->ctrl->num_sms * 2u; }
inline size_t kv_parts_at(uint32_t workers) { return (sizeof(kv_launch_words_t) + 4 * (size_t)workers + 127) / 128 * 128; }

/* The attention's launchers, one translation unit per element type. */
template <class T>
int kv_launch_attend(bam_array* a, const kv_layout_d_t& L, const bam_kv_attend_t* p, void* scratch, void* stream);
extern template int kv_launch_attend<__nv_bfloat16>(bam_array*, const kv_layout_d_t&, const bam_kv_attend_t*, void*, void*);
extern template int kv_launch_attend<__half>(bam_array*, const kv_layout_d_t&, const bam_kv_attend_t*, void*, void*);

}  // namespace bam
#endif
