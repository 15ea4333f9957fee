// The exact paged cache: what its kernels share.  A page holds `page` tokens of every kv head as 16-bit key and value rows;
// element (block, token, head, :) of a plane is at block * sb + token * st + head * sh (bytes here), rows 16-byte aligned.
#pragma once
#include "tq_common.cuh"

namespace tqpg {

// Quotients of numbers below 2^31 by a number that the host knows: q = n * mul >> (31 + shift), exact for mul = ceil(2^(31 + shift) / d)
// with 2^shift >= d, since the excess of mul is below 2^shift / 2^(31 + shift) a unit of n.
struct Divisor {
    uint32_t mul;
    int shift, d;
    __device__ __forceinline__ int quotient(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> (31 + shift)); }
};
inline Divisor divisor(int d) {
    int s = 0;
    while (((int64_t)1 << s) < d) ++s;
    return Divisor{(uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), s, d};
}

struct Pages {
    uint8_t* k;
    uint8_t* v;
    int64_t num_blocks;
    int64_t sb, st, sh;   // bytes
    int page, H;
    Divisor by_page;
};
struct Batch {
    const int32_t* table;
    const int32_t* lens;
    int table_stride, batch, max_seq_len;
    const int32_t *held, *seen;    // of a ledger, or NULL
};

// Longest table index a length may reach is checked on the host (max_seq_len against the table's width); a length outside
// [0, max_seq_len] is clamped and reported.
__device__ __forceinline__ int seq_len(const Batch& q, int b, int32_t* status) {
    const int n = q.lens[b];
    if (n >= 0 && n <= q.max_seq_len) return n;
    atomicCAS(status, 0, (int)TQ_ERR_RANGE);
    return n < 0 ? 0 : q.max_seq_len;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes to shared memory, zeros where `ok` is false (nothing is read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Launch as a programmatic dependent: the CTAs may take their places while the launch ahead finishes.  Every kernel launched so
// waits for it before it reads or writes anything, and lets the launch behind begin only after that, with one exception: the
// second launch of an observation reads lengths, tables, queries and keys (and may note an error) before its wait.  It directly
// follows the first one, which writes none of those and has waited for everything ahead before this one may begin.
template <class... P, class... A>
inline int launch_behind_as(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess ? TQ_OK : TQ_ERR_CUDA;
}
template <class... P, class... A>
inline int launch_behind(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    return launch_behind_as(kernel, grid, threads, smem, 1, st, args...);
}
template <class... P, class... A>
inline int launch_behind_in_clusters(void (*kernel)(P...), dim3 grid, int threads, int cluster, cudaStream_t st, A... args) {
    return launch_behind_as(kernel, grid, threads, 0, cluster, st, args...);
}

inline int pages_check(const tq_pages* g) {
    if (!g || !g->key || !g->value) return TQ_ERR_NULL;
    if (g->head_dim != 64 && g->head_dim != 128 && g->head_dim != 256) return TQ_ERR_UNSUPPORTED;
    if (g->dtype != TQ_BF16 && g->dtype != TQ_F16) return TQ_ERR_UNSUPPORTED;
    if (g->num_blocks < 1 || g->block_size < 1 || g->num_kv_heads < 1 || g->num_kv_heads > 65535) return TQ_ERR_SHAPE;
    if (g->num_blocks >= ((int64_t)1 << 31)) return TQ_ERR_SHAPE;
    if (((uintptr_t)g->key & 15) || ((uintptr_t)g->value & 15) || (g->stride_block & 7) || (g->stride_token & 7) || (g->stride_head & 7))
        return TQ_ERR_ALIGN;
    if (g->stride_block < 0 || g->stride_token < 0 || g->stride_head < 0) return TQ_ERR_SHAPE;
    return TQ_OK;
}
inline Pages pages_of(const tq_pages* g) {
    return Pages{static_cast<uint8_t*>(g->key), static_cast<uint8_t*>(g->value), g->num_blocks, g->stride_block * 2,
                 g->stride_token * 2, g->stride_head * 2, g->block_size, g->num_kv_heads, divisor(g->block_size)};
}
// What a list of work (units of a decode, tiles of an observation) may hold: its indices, rounded up to shares, stay below 2^31.
constexpr int64_t MAX_UNITS = ((int64_t)1 << 31) - (1 << 20);
// A table row covers max_seq_len tokens.
inline int batch_check(const tq_pages* g, const tq_pages_batch* q) {
    if (!q || !q->block_tables || !q->seq_lens || !q->held != !q->seen) return TQ_ERR_NULL;
    if (q->batch < 1 || q->max_seq_len < 1 || q->table_width < 1 || q->table_stride < q->table_width) return TQ_ERR_SHAPE;
    if ((int64_t)q->table_width * g->block_size < q->max_seq_len || q->max_seq_len > (1 << 30)) return TQ_ERR_RANGE;
    return TQ_OK;
}
inline Batch batch_of(const tq_pages_batch* q) {
    return Batch{q->block_tables, q->seq_lens, q->table_stride, q->batch, q->max_seq_len, q->held, q->seen};
}

}  // namespace tqpg
