/* bam_kv_attend_bf16.cu -- the attention kernels for __nv_bfloat16 rows (see bam_kv_attend.cuh) */
#include "bam_kv_attend.cuh"

template int bam::kv_launch_attend<__nv_bfloat16>(bam_array*, const bam::kv_layout_d_t&, const bam_kv_attend_t*, void*, void*);
