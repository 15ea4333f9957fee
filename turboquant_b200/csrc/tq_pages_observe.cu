// The weights of a prompt's last queries over the exact paged cache, without their output: what each cached token receives.
//
// Rows r = (query i of the window, query head of the kv head's group), R = window * G of them:
//     s_rt = scale <q_r, k_t>,  t <= n - window + i(r);   lse_r = log2 sum_t 2^(s_rt);   mass_t += sum_r 2^(s_rt - lse_r)
// (s in the log2 domain).  lse needs every key before the first weight is known, so the keys are gone over twice: the first launch
// keeps a running maximum and sum per row and split, the second forms the weights.  Both are products of 128 x 128 tiles on the
// 5th-generation tensor cores, turned so that what is summed lies in one thread: queries in the rows (tensor-memory lanes) of the
// first, whose threads sum along the keys, tokens in the rows of the second, whose threads sum along the queries.
//
// A CTA walks tiles of 128 tokens: copies of tile i + 1, the product of tile i and the exponentials of tile i - 1 run at the same
// time.  Key tiles lie in shared memory as the tensor cores want them (64 channels a box, 128-byte swizzle), brought by 16-byte
// asynchronous copies through the block table, so that a page may end anywhere.
#include "tq_pages.cuh"
#include "tq_tcgen05.cuh"

using namespace tqpg;
using namespace tqtc;

namespace {

constexpr int OB_TILE = 128, OB_THREADS = 256, OB_BOX = OB_TILE * 128;

struct ObserveParams {
    Pages g;
    Batch q;
    const uint8_t* query;     // (batch, window, Qh, D)
    int Qh, G, window, R;     // R = window * G
    int row_tiles, splits;
    float scale_log2;
    int is_bf16;
    float2* stats;            // [batch * H][row tile][split][half][128] (maximum, sum) of a row
    float* mass;
    int64_t mass_stride;
    int32_t* status;
};

// at least 80 KB, so that no more than two CTAs, with 256 columns of tensor memory each, meet on an SM
template <int D>
constexpr size_t observe_smem() { return D == 64 ? (size_t)80 * 1024 : (size_t)3 * (D / 64) * OB_BOX + 1024; }

// SECOND: the launch that forms the weights
template <int D, bool SECOND>
__global__ void __launch_bounds__(OB_THREADS, 1) tq_pages_observe_kernel(const ObserveParams p) {
    constexpr int BOXES = D / 64, TILE_BYTES = BOXES * OB_BOX;
    constexpr int LPR = D / 8, RPI = OB_THREADS / LPR, ITER = OB_TILE / RPI;      // lanes a row, rows a step, steps a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (tq_smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sQ = smem, *sK = smem + TILE_BYTES;                                   // [2] key tiles
    __shared__ uint64_t bars[2];
    __shared__ uint32_t s_tmem;
    __shared__ uint8_t s_there[4][OB_TILE];                                        // the token's page exists
    __shared__ float s_lse[OB_TILE], s_part[OB_TILE];

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, half = w >> 2;
    const int pair = SECOND ? blockIdx.y : blockIdx.z, b = pair / p.g.H, h = pair % p.g.H;
    const int n = seq_len(p.q, b, p.status);
    const int tiles = (n + OB_TILE - 1) / OB_TILE, per = (tiles + p.splits - 1) / p.splits;
    const int first = blockIdx.x * per, count = min(per, tiles - first);           // this CTA's tiles
    if (n == 0 || (SECOND && count <= 0)) return;

    auto stats_at = [&](int rt, int split, int hf) {
        return p.stats + ((((int64_t)pair * p.row_tiles + rt) * p.splits + split) * 2 + hf) * OB_TILE;
    };
    if (!SECOND && count <= 0) {                                                   // no tiles: an empty sum
        stats_at(blockIdx.y, blockIdx.x, half)[tid & 127] = make_float2(-INFINITY, 0.f);
        return;
    }

    if (w == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tq_smem_u32(&s_tmem)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        tq_mbar_init(bars, 1);
        tq_mbar_init(bars + 1, 1);
        tq_mbar_fence_init();
    }

    const int r0 = tid / LPR, ch = tid % LPR;
    const uint32_t col = (ch >> 3) * OB_BOX;                                       // box of this lane's 16 bytes
    auto swizzled = [&](int r) { return col + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
    const int32_t* table = p.q.table + (int64_t)b * p.q.table_stride;
    int entries[ITER];
    auto look_up = [&](int tile) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int t = (first + tile) * OB_TILE + i * RPI + r0;
            entries[i] = tile < count && t < n ? table[t / p.g.page] : -1;
        }
    };
    auto load_tile = [&](int tile) {                                               // with the entries looked up for it
        const uint32_t dst = tq_smem_u32(sK) + (tile & 1) * TILE_BYTES;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int r = i * RPI + r0, t = (first + tile) * OB_TILE + r, e = entries[i];
            const bool ok = tile < count && t < n && (uint32_t)e < (uint64_t)p.g.num_blocks;
            if (!ok && tile < count && t < n && ch == 0) atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
            const int64_t off = ok ? e * p.g.sb + (t % p.g.page) * p.g.st + h * p.g.sh + ch * 16 : 0;
            if (tile < count) cp_async16(dst + swizzled(r), p.g.k + off, ok);
            if (ch == 0 && tile < count) s_there[tile & 3][r] = ok;
        }
        cp_async_commit();
    };
    auto load_rows = [&](int rt) {                                                 // query rows, zeros behind the last
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int r = i * RPI + r0, row = rt * OB_TILE + r;
            const bool ok = row < p.R;
            const int64_t off = ok ? ((((int64_t)b * p.window + row / p.G) * p.Qh + h * p.G + row % p.G) * D + ch * 8) * 2 : 0;
            cp_async16(tq_smem_u32(sQ) + swizzled(r), p.query + off, ok);
        }
    };
    auto elected = [&]() -> bool {
        uint32_t pred;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
        return pred != 0;
    };

    const int rt_from = SECOND ? 0 : blockIdx.y, rt_to = SECOND ? p.row_tiles : blockIdx.y + 1;
    uint32_t phase[2] = {0u, 0u};
    bool failed = false;
#pragma unroll 1
    for (int rt = rt_from; rt < rt_to && !failed; ++rt) {
        const int rows = min(OB_TILE, p.R - rt * OB_TILE);
        const uint32_t cols = SECOND ? (uint32_t)(rows + 15) / 16 * 16 : (uint32_t)OB_TILE;
        const uint32_t idesc = umma_idesc_bf16(cols, false, !p.is_bf16);
        load_rows(rt);
        look_up(0);
        load_tile(0);
        look_up(1);
        load_tile(1);
        if (SECOND && tid < OB_TILE) {                                             // the rows' sums over all splits
            float m = -INFINITY, l = 0.f;
            if (tid < rows) {
#pragma unroll 4
                for (int s = 0; s < 2 * p.splits; ++s) m = fmaxf(m, stats_at(rt, s >> 1, s & 1)[tid].x);
#pragma unroll 4
                for (int s = 0; s < 2 * p.splits; ++s) {
                    const float2 v = stats_at(rt, s >> 1, s & 1)[tid];
                    if (v.x != -INFINITY) l += v.y * ex2(v.x - m);
                }
            }
            s_lse[tid] = l == 0.f ? INFINITY : m + log2f(l);
        }
        // first launch: row of this thread and the last token it sees; second: token of this thread
        const int lane_row = (w & 3) * 32 + lane;
        const int last = SECOND ? 0 : n - p.window + (rt * OB_TILE + lane_row) / p.G;
        float m = -INFINITY, l = 0.f;
        bool bad = false;
#pragma unroll 1
        for (int i = 0; i <= count; ++i) {
            if (i < count) {
                if (i == 0) cp_async_wait<1>();                                    // the second tile may still be under way
                else cp_async_wait<0>();
                tq_fence_proxy_async();
            }
            tc_fence_before();
            if (__syncthreads_or(bad)) {
                failed = true;
                break;
            }
            tc_fence_after();
            if (i < count && w == 0) {
                const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0) + (i & 1) * 128;
                if (elected()) {
                    const uint32_t aQ = tq_smem_u32(sQ), aK = tq_smem_u32(sK) + (i & 1) * TILE_BYTES;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = (ks >> 2) * OB_BOX + (ks & 3) * 32;
                        if (SECOND) umma_ss(tmem, smem_desc_sw128(aK + off), smem_desc_sw128(aQ + off), idesc, ks ? 1u : 0u);
                        else umma_ss(tmem, smem_desc_sw128(aQ + off), smem_desc_sw128(aK + off), idesc, ks ? 1u : 0u);
                    }
                    umma_commit(bars + (i & 1));
                }
                __syncwarp();
            }
            if (i == 0) continue;
            const int j = i - 1;                                                   // the tile whose product is looked at
            if (!tq_mbar_wait_bounded(bars + (j & 1), phase[j & 1], 1 << 22)) bad = true;
            phase[j & 1] ^= 1u;
            tc_fence_after();
            if (i + 1 < count) {                                                   // its stage is free
                look_up(i + 1);
                load_tile(i + 1);
            }
            const uint32_t base = s_tmem + ((uint32_t)((w & 3) * 32) << 16) + (j & 1) * 128;
            const int t0 = (first + j) * OB_TILE;
            const uint8_t* there = s_there[j & 3];
            if (!SECOND) {
                if ((w & 3) * 32 < rows) {                                         // rows behind the last: nothing to do for the warp
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int c0 = half * 64 + c * 32;
                        float s[32];
                        tmem_ld32(base + c0, s);
                        const int see = last - t0 - c0;                            // columns 0 .. see
                        const bool gone = there[c0 + lane] == 0;
                        if (__any_sync(0xffffffffu, gone || see < 31)) {
                            const uint32_t out = __ballot_sync(0xffffffffu, gone);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (k > see || ((out >> k) & 1)) s[k] = -INFINITY;
                        }
                        float mx = s[0] * p.scale_log2;
                        s[0] = mx;
#pragma unroll
                        for (int k = 1; k < 32; ++k) {
                            s[k] *= p.scale_log2;
                            mx = fmaxf(mx, s[k]);
                        }
                        if (mx > m) {
                            l *= m == -INFINITY ? 0.f : ex2(m - mx);
                            m = mx;
                        }
                        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                        for (int k = 0; k < 32; ++k) l += ex2(s[k] - ref);
                    }
                }
            } else {
                const int t = t0 + lane_row;
                // query i sees token t from i = t - (n - window) on
                const int from = max(0, (t - n + p.window)) * p.G - rt * OB_TILE;
                float sum = 0.f;
                for (int c0 = half * 32; c0 < rows; c0 += 64) {
                    float s[32];
                    tmem_ld32(base + c0, s);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float e = ex2(s[k] * p.scale_log2 - s_lse[c0 + k]);
                        sum += c0 + k >= from && c0 + k < rows ? e : 0.f;
                    }
                }
                if (half == 1) s_part[lane_row] = sum;
                __syncthreads();
                if (half == 0 && t < n && there[lane_row]) p.mass[pair * p.mass_stride + t] += sum + s_part[lane_row];
            }
        }
        if (!SECOND) stats_at(rt, blockIdx.x, half)[lane_row] = make_float2(m, l);
        if (__syncthreads_or(bad)) failed = true;                                  // the next row tile takes the buffers over
    }
    if (failed && tid == 0) atomicCAS(p.status, 0, (int)TQ_ERR_TIMEOUT);
    cp_async_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (w == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(256) : "memory");
}

struct Plan {
    int row_tiles, splits;
    size_t bytes;
};
// Two CTAs' worth of work for every SM, as far as the longest sequence has tiles.
Plan plan_of(const tq_pages* g, const tq_pages_batch* q, int window, int Qh) {
    Plan s;
    const int64_t R = (int64_t)window * (Qh / g->num_kv_heads), pairs = (int64_t)q->batch * g->num_kv_heads;
    s.row_tiles = (int)((R + OB_TILE - 1) / OB_TILE);
    const int64_t tiles = ((int64_t)q->max_seq_len + OB_TILE - 1) / OB_TILE, want = 4 * tq_sm_count() / (pairs * s.row_tiles) + 1;
    s.splits = (int)(want < tiles ? want : tiles);
    s.bytes = (size_t)pairs * s.row_tiles * s.splits * 2 * OB_TILE * sizeof(float2);
    return s;
}
int observe_check(const tq_pages* g, const tq_pages_batch* q, int window, int Qh) {
    int rc = pages_check(g);
    if (rc == TQ_OK) rc = batch_check(g, q);
    if (rc != TQ_OK) return rc;
    if (window < 1 || Qh < 1 || Qh % g->num_kv_heads != 0) return TQ_ERR_SHAPE;
    if ((int64_t)window * (Qh / g->num_kv_heads) > (1 << 20) || (int64_t)q->batch * g->num_kv_heads > 65535) return TQ_ERR_SHAPE;
    return TQ_OK;
}
template <int D>
int launch(const ObserveParams& p, cudaStream_t st) {
    static TqSmemOptIn opt_a, opt_b;
    if (tq_opt_in_smem(tq_pages_observe_kernel<D, false>, observe_smem<D>(), opt_a) != TQ_OK ||
        tq_opt_in_smem(tq_pages_observe_kernel<D, true>, observe_smem<D>(), opt_b) != TQ_OK)
        return TQ_ERR_CUDA;
    const unsigned pairs = (unsigned)(p.q.batch * p.g.H);
    tq_pages_observe_kernel<D, false><<<dim3((unsigned)p.splits, (unsigned)p.row_tiles, pairs), OB_THREADS, observe_smem<D>(), st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return TQ_ERR_CUDA;
    tq_pages_observe_kernel<D, true><<<dim3((unsigned)p.splits, pairs), OB_THREADS, observe_smem<D>(), st>>>(p);
    return cudaGetLastError() == cudaSuccess ? TQ_OK : TQ_ERR_CUDA;
}

}  // namespace

extern "C" int tq_pages_observe_scratch_bytes(const tq_pages* pages, const tq_pages_batch* batch, int32_t window, int32_t num_q_heads,
                                              size_t* out) {
    if (!out) return TQ_ERR_NULL;
    const int rc = observe_check(pages, batch, window, num_q_heads);
    if (rc != TQ_OK) return rc;
    *out = plan_of(pages, batch, window, num_q_heads).bytes;
    return TQ_OK;
}

extern "C" int tq_pages_observe(const tq_pages* pages, const tq_pages_batch* batch, const void* query, int32_t window, int32_t num_q_heads,
                                float scale, float* mass, int64_t mass_stride, void* scratch, size_t scratch_bytes, int32_t* status,
                                void* stream) {
    const int rc = observe_check(pages, batch, window, num_q_heads);
    if (rc != TQ_OK) return rc;
    if (!query || !mass || !scratch || !status) return TQ_ERR_NULL;
    if (((uintptr_t)query & 15) || ((uintptr_t)scratch & 15)) return TQ_ERR_ALIGN;
    if (mass_stride < batch->max_seq_len) return TQ_ERR_RANGE;
    const Plan s = plan_of(pages, batch, window, num_q_heads);
    if (scratch_bytes < s.bytes) return TQ_ERR_WORKSPACE;
    ObserveParams p;
    p.g = pages_of(pages);
    p.q = batch_of(batch);
    p.query = static_cast<const uint8_t*>(query);
    p.Qh = num_q_heads;
    p.G = num_q_heads / pages->num_kv_heads;
    p.window = window;
    p.R = window * p.G;
    p.row_tiles = s.row_tiles;
    p.splits = s.splits;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.is_bf16 = pages->dtype == TQ_BF16;
    p.stats = static_cast<float2*>(scratch);
    p.mass = mass;
    p.mass_stride = mass_stride;
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    tq_note_launch(st, TQ_LAUNCH_WAITED);
    switch (pages->head_dim) {
        case 64: return launch<64>(p, st);
        case 128: return launch<128>(p, st);
        default: return launch<256>(p, st);
    }
}
