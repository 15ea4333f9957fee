// The weights of a prompt's last queries over the exact paged cache, without their output: what each cached token receives.
//
// Rows r = (query i of the window, query head of the kv head's group), R = window * G of them:
//     s_rt = scale <q_r, k_t>,  t <= n - window + i(r);   lse_r = log2 sum_t 2^(s_rt);   mass_t += sum_r 2^(s_rt - lse_r)
// (s in the log2 domain).  lse needs every key before the first weight is known, so the keys are gone over twice (for every 128
// rows): the first launch keeps a running maximum and sum per row and split, the second forms the weights.  Both are products of
// 128 x 128 tiles on the 5th-generation tensor cores, turned so that what is summed lies in one thread: queries in the rows
// (tensor-memory lanes) of the first, whose threads sum along the keys, tokens in the rows of the second, whose threads sum along
// the queries.
//
// The tiles (128 tokens of one kv head of one sequence) of a batch are one list in the order sequence, head, row tile, token, of
// which every CTA, two an SM, takes an equal share.  In a share, copies of tile i + 1, the product of tile i and the exponentials
// of tile i - 1 run at the same time.  Key tiles lie in shared memory as the tensor cores want them (64 channels a box, 128-byte
// swizzle), brought by 16-byte asynchronous copies through the block table, so that a page may end anywhere.
//
// Measured: 16 queries of 8 sequences of 4096 to 32768, 32 / 8 heads of 128: 156 us for two times 291 MB.  Copies alone take 54 us
// a launch, products and exponentials alone 44; the rest is their hand-over (a barrier of the CTA for every tile, two in the second
// launch; no unit is busy for half of the time).  32 queries of one prompt of 5003: 19 us.
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
    int Qh, window, R;        // R = window * G
    Divisor by_group;         // G, query heads per kv head
    int row_tiles;
    float scale_log2;
    int is_bf16;
    float2* stats;            // [(sequence, head, row tile) + CTA][128]: maximum and sum of a row over the CTA's tiles
    float* mass;
    int64_t mass_stride;
    int32_t* status;
};

// at least 80 KB, so that no more than two CTAs, with 256 columns of tensor memory each, meet on an SM
template <int D>
constexpr size_t observe_smem() { return D == 64 ? (size_t)80 * 1024 : (size_t)3 * (D / 64) * OB_BOX + 1024; }

__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves_of(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// 2^(x - top) of a piece's maximum x, 1 where it is the largest: sums that are NaN under a maximum of -inf (scores that are all NaN) stay NaN
__device__ __forceinline__ float share_of_top(float x, float top) { return x == top ? 1.f : ex2(x - top); }

// A length as it lies in the second-level cache: the second launch asks before it waits for the first one, which has waited for
// everything ahead of it.
__device__ __forceinline__ int fresh_len(const Batch& q, int b, int32_t* status) {
    const int n = __ldcg(q.lens + b);
    if (n >= 0 && n <= q.max_seq_len) return n;
    atomicCAS(status, 0, (int)TQ_ERR_RANGE);
    return n < 0 ? 0 : q.max_seq_len;
}

// SECOND: the launch that forms the weights
template <int D, bool SECOND>
__global__ void __launch_bounds__(OB_THREADS, D == 256 ? 1 : 2) tq_pages_observe_kernel(const ObserveParams p) {
    constexpr int BOXES = D / 64, TILE_BYTES = BOXES * OB_BOX;
    constexpr int LPR = D / 8, RPI = OB_THREADS / LPR, ITER = OB_TILE / RPI;      // lanes a row, rows a step, steps a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (tq_smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sQ = smem, *sK = smem + TILE_BYTES;                                   // [2] key tiles
    __shared__ uint64_t bars[2];
    __shared__ uint32_t s_tmem;
    __shared__ int64_t s_off[4][OB_TILE];                                          // rows of a tile in the key plane, -1: no such page
    __shared__ float2 s_stat[OB_THREADS];
    __shared__ float s_lse[OB_TILE], s_part[OB_TILE];
    __shared__ int s_sum[8], s_at[3];

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, half = w >> 2;
    if (!SECOND) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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

    // ---- this CTA's share of the list.  The second launch forms all row tiles of a token tile one after the other; its list has
    // no row tiles of its own.
    const int per_seq_first = p.g.H * p.row_tiles, per_seq = SECOND ? p.g.H : per_seq_first;      // lists a sequence's tiles come in
    auto tiles_of = [&](int b) { return b < p.q.batch ? (fresh_len(p.q, b, p.status) + OB_TILE - 1) / OB_TILE : 0; };
    auto scan = [&](int c, int& total) {
        int x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_sum[w] = x;
        __syncthreads();
        total = 0;
        int before = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < w) before += s_sum[i];
            total += s_sum[i];
        }
        __syncthreads();
        return x + before;
    };
    const int c0 = tiles_of(tid);
    int all = 0, incl0 = 0, total0 = 0;
    for (int b0 = 0; b0 < p.q.batch; b0 += OB_THREADS) {
        int total;
        const int incl = scan(b0 == 0 ? c0 : tiles_of(b0 + tid), total);
        if (b0 == 0) incl0 = incl, total0 = total;
        all += total;
    }
    auto share_for = [&](int lists) { return max(1, (int)(((int64_t)all * lists + gridDim.x - 1) / gridDim.x)); };
    const int share_first = share_for(per_seq_first), share = share_for(per_seq), T = all * per_seq;
    const int lo = (int)min((int64_t)T, (int64_t)blockIdx.x * share), n_tiles = min(T - lo, share);
    for (int b0 = 0, carry = 0; b0 < p.q.batch; b0 += OB_THREADS) {
        const int c = b0 == 0 ? c0 : tiles_of(b0 + tid);
        int total = total0;
        const int incl = b0 == 0 ? incl0 : scan(c, total), from = (carry + incl - c) * per_seq;
        if (lo >= from && lo < from + c * per_seq) {
            s_at[0] = b0 + tid;
            s_at[1] = from;
            s_at[2] = (carry + incl - c) * per_seq_first;
        }
        carry += total;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    const int r0 = tid / LPR, ch = tid % LPR;
    const uint32_t in_box = (ch >> 3) * OB_BOX + r0 * 128;                         // of this lane's 16 bytes in its first row
    auto swizzled = [&](int i) { return in_box + i * RPI * 128 + (((ch & 7) ^ ((i * RPI + r0) & 7)) << 4); };
    auto elected = [&]() -> bool {
        uint32_t pred;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
        return pred != 0;
    };
    const int lane_row = (w & 3) * 32 + lane;                                      // tensor-memory lane of this thread
    // First launch, up to 64 rows: the query tile holds every row twice, so that all four parts of the SM have exponentials to do;
    // a thread then sums a quarter of a tile's keys in the place of half of them.
    const bool twice = !SECOND && p.R <= 64;
    uint32_t phase[2] = {0u, 0u};
    bool failed = false, waited = !SECOND;
    int done = 0;
    int b = n_tiles > 0 ? s_at[0] : 0, base_first = n_tiles > 0 ? s_at[2] : 0;     // base_first: where sequence b begins in the first launch's list
    int list = 0, tile0 = 0, n = 0, tiles = 0;
    int ordered = 0;                                                               // the slot from which on slots are in the sequence's order
    auto begin = [&]() {                                                           // sequence b
        n = fresh_len(p.q, b, p.status);
        tiles = (n + OB_TILE - 1) / OB_TILE;
        const int held = p.q.held != nullptr ? __ldcg(p.q.held + b) : 0;
        ordered = held > 0 && __ldcg(p.q.seen + b) != held ? held : 0;
        if (ordered > max(0, n - p.window) && tid == 0 && n > 0) atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
    };
    if (n_tiles > 0) {
        begin();
        const int rel = lo - s_at[1];
        list = rel / tiles;
        tile0 = rel - list * tiles;
    }
#pragma unroll 1
    while (done < n_tiles && !failed) {
        // ---- tiles [tile0, tile0 + count) of one (sequence, kv head)
        const int count = min(tiles - tile0, n_tiles - done);
        const int h = SECOND ? list : list / p.row_tiles;
        const int32_t* table = p.q.table + (int64_t)b * p.q.table_stride;
        const int64_t head_off = h * p.g.sh;
        int entry = 0;
        auto look_up = [&](int i) {                                                // page of this thread's row of tile i, asked for early
            const int t = (tile0 + i) * OB_TILE + tid;
            entry = tid < OB_TILE && i < count && t < n ? __ldcg(table + p.g.by_page.quotient(t)) : -1;
        };
        auto note_row = [&](int i) {
            const int t = (tile0 + i) * OB_TILE + tid;
            if (tid < OB_TILE && i < count) {
                const bool ok = (uint32_t)entry < (uint64_t)p.g.num_blocks;
                if (!ok && t < n) atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
                s_off[i & 3][tid] = ok ? entry * p.g.sb + (int64_t)(t - p.g.by_page.quotient(t) * p.g.page) * p.g.st + head_off : -1;
            }
        };
        auto load_tile = [&](int i) {
            if (i < count) {
                const uint32_t dst = tq_smem_u32(sK) + (i & 1) * TILE_BYTES;
                const uint8_t* k = p.g.k + ch * 16;
#pragma unroll
                for (int j = 0; j < ITER; ++j) {
                    const int64_t off = s_off[i & 3][j * RPI + r0];
                    cp_async16(dst + swizzled(j), k + (off < 0 ? 0 : off), off >= 0);
                }
            }
            cp_async_commit();
        };
        const int rt_from = SECOND ? 0 : list - h * p.row_tiles, rt_to = SECOND ? p.row_tiles : rt_from + 1;
#pragma unroll 1
        for (int rt = rt_from; rt < rt_to && !failed; ++rt) {
            const int rows = min(OB_TILE, p.R - rt * OB_TILE);
            const uint32_t cols = SECOND ? (uint32_t)(rows + 15) / 16 * 16 : (uint32_t)OB_TILE;
            const uint32_t idesc = umma_idesc_bf16(cols, false, !p.is_bf16);
            look_up(0);
            const int entry0 = entry;
            look_up(1);
            const int entry1 = entry;
            entry = entry0;
            note_row(0);
            entry = entry1;
            note_row(1);
#pragma unroll
            for (int j = 0; j < ITER; ++j) {                                       // query rows, zeros behind the last
                const int r = j * RPI + r0, row = rt * OB_TILE + (twice ? r & 63 : r), i = p.by_group.quotient(row);
                const bool ok = row < p.R;
                const int64_t off = ok ? ((((int64_t)b * p.window + i) * p.Qh + h * p.by_group.d + row - i * p.by_group.d) * D + ch * 8) * 2 : 0;
                cp_async16(tq_smem_u32(sQ) + swizzled(j), p.query + off, ok);
            }
            __syncthreads();
            load_tile(0);
            load_tile(1);
            look_up(2);
            if (SECOND) {                                                          // the rows' sums over all of the first launch's pieces
                if (!waited) {
                    asm volatile("griddepcontrol.wait;" ::: "memory");
                    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
                    waited = true;
                }
                const int begin = base_first + (h * p.row_tiles + rt) * tiles;
                const int from = begin / share_first, to = (begin + tiles - 1) / share_first;
                const float2* st = p.stats + ((int64_t)(b * p.g.H + h) * p.row_tiles + rt) * OB_TILE + (tid & 127);
                float m = -INFINITY, l = 0.f;
#pragma unroll 1
                for (int k0 = from + half; k0 <= to; k0 += 16) {                   // a thread every other piece
                    float2 v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = k0 + 2 * k <= to ? __ldcg(st + (int64_t)(k0 + 2 * k) * OB_TILE) : make_float2(-INFINITY, 0.f);
                    float mx = m;
#pragma unroll
                    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, v[k].x);
                    l *= share_of_top(m, mx);
                    m = mx;
#pragma unroll
                    for (int k = 0; k < 8; ++k) l = fmaf(v[k].y, share_of_top(v[k].x, mx), l);
                }
                s_stat[tid] = make_float2(m, l);
                __syncthreads();
                if (tid < OB_TILE) {
                    const float2 o = s_stat[tid + OB_TILE];
                    const float mx = fmaxf(m, o.x);
                    const float sum = l * share_of_top(m, mx) + o.y * share_of_top(o.x, mx);
                    s_lse[tid] = sum == 0.f || tid >= rows ? INFINITY : mx + log2f(sum);
                }
            }
            // first launch: the last token that this thread's row sees
            const int my_row = twice ? lane_row & 63 : lane_row;
            const int at = SECOND ? 0 : n - p.window + p.by_group.quotient(rt * OB_TILE + my_row), last = at < ordered ? -1 : at;
            float m = -INFINITY, l = 0.f;
            bool bad = false;
#pragma unroll 1
            for (int i = 0; i <= count; ++i) {
                if (i > 0 && i + 1 < count) note_row(i + 1);
                if (i < count) {
                    if (i == 0) cp_async_wait<1>();                                // the second tile may still be under way
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
                const int j = i - 1;                                               // the tile whose product is looked at
                if (!tq_mbar_wait_bounded(bars + (j & 1), phase[j & 1], 1 << 22)) bad = true;
                phase[j & 1] ^= 1u;
                tc_fence_after();
                if (i + 1 < count) {                                               // its stage is free
                    load_tile(i + 1);
                    look_up(i + 2);
                }
                const uint32_t base = s_tmem + ((uint32_t)((w & 3) * 32) << 16) + (j & 1) * 128;
                const int t0 = (tile0 + j) * OB_TILE;
                const int64_t* there = s_off[j & 3];
                if (!SECOND) {
                    if (twice || (w & 3) * 32 < rows) {                            // rows behind the last: nothing to do for the warp
#pragma unroll 1
                        for (int c = 0; c < (twice ? 1 : 2); ++c) {
                            const int col = twice ? half * 64 + (lane_row >> 6) * 32 : half * 64 + c * 32;
                            float s[32];
                            tmem_ld32(base + col, s);
                            const int see = last - t0 - col;                       // columns 0 .. see
                            const bool gone = there[col + lane] < 0;
                            float scale = p.scale_log2;
                            if (__any_sync(0xffffffffu, gone || see < 31)) {
                                const uint32_t out = __ballot_sync(0xffffffffu, gone);
#pragma unroll
                                for (int k = 0; k < 32; ++k) s[k] = k > see || ((out >> k) & 1) ? -INFINITY : s[k] * scale;
                                scale = 1.f;
                            }
                            float top = max3(s[0], s[1], s[2]);
                            if (scale < 0.f) {                                     // the largest scaled score belongs to the smallest
                                top = s[0];
#pragma unroll
                                for (int k = 1; k < 32; ++k) top = fminf(top, s[k]);
                            } else {
#pragma unroll
                                for (int k = 3; k + 1 < 32; k += 2) top = max3(top, s[k], s[k + 1]);
                                top = fmaxf(top, s[31]);
                            }
                            const float mx = top * scale;
                            if (mx > m) {
                                l *= ex2(m - mx);                                  // zero times 2^-inf at first
                                m = mx;
                            }
                            const float ref = m == -INFINITY ? 0.f : -m;
                            const uint64_t scale2 = pair_of(scale, scale), ref2 = pair_of(ref, ref);
                            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const float2 x = halves_of(fma_pair(pair_of(s[2 * k], s[2 * k + 1]), scale2, ref2));
                                sum2[k & 1] = add_pair(sum2[k & 1], pair_of(ex2(x.x), ex2(x.y)));
                            }
                            const float2 sum = halves_of(add_pair(sum2[0], sum2[1]));
                            l += sum.x + sum.y;
                        }
                    }
                } else {
                    const int t = t0 + lane_row;
                    // query i sees token t from i = t - (n - window) on, if it lies in the part that is in order
                    const int from = min(max(0, max(t, ordered) - n + p.window), p.window) * p.by_group.d - rt * OB_TILE;
                    const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2);
                    uint64_t sum2[2] = {0ull, 0ull};
                    float sum = 0.f;
#pragma unroll 1
                    for (int col = half * 32; col < rows; col += 64) {
                        float s[32];
                        tmem_ld32(base + col, s);
                        if (__any_sync(0xffffffffu, from > col) || col + 32 > rows) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                const float e = ex2(s[k] * p.scale_log2 - s_lse[col + k]);
                                sum += col + k >= from && col + k < rows ? e : 0.f;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const float2 lse = *reinterpret_cast<const float2*>(s_lse + col + 2 * k);
                                const float2 x = halves_of(fma_pair(pair_of(s[2 * k], s[2 * k + 1]), scale2, pair_of(-lse.x, -lse.y)));
                                sum2[k & 1] = add_pair(sum2[k & 1], pair_of(ex2(x.x), ex2(x.y)));
                            }
                        }
                    }
                    const float2 both = halves_of(add_pair(sum2[0], sum2[1]));
                    sum += both.x + both.y;
                    if (half == 1) s_part[lane_row] = sum;
                    __syncthreads();
                    if (half == 0 && t < n && there[lane_row] >= 0) p.mass[(int64_t)(b * p.g.H + h) * p.mass_stride + t] += sum + s_part[lane_row];
                }
            }
            if (!SECOND) {                                                         // the parts of a row, then its piece of the statistics
                s_stat[tid] = make_float2(m, l);
                __syncthreads();
                if (tid < (twice ? 64 : OB_TILE)) {
                    float mx = m, sum = 0.f;
                    for (int k = tid; k < OB_THREADS; k += twice ? 64 : OB_TILE) mx = fmaxf(mx, s_stat[k].x);
                    for (int k = tid; k < OB_THREADS; k += twice ? 64 : OB_TILE) sum = fmaf(s_stat[k].y, share_of_top(s_stat[k].x, mx), sum);
                    p.stats[(((int64_t)(b * p.g.H + h) * p.row_tiles + rt) + blockIdx.x) * OB_TILE + tid] = make_float2(mx, sum);
                }
            }
            if (__syncthreads_or(bad)) failed = true;                              // whoever comes next takes the buffers over
        }
        done += count;
        tile0 = 0;
        if (done < n_tiles && ++list == per_seq) {
            list = 0;
            do {
                base_first += tiles * per_seq_first;
                ++b;
                begin();
            } while (n == 0 && b + 1 < p.q.batch);                                 // a share ends with its last tile: there is one ahead
        }
    }
    if (SECOND && !waited) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    if (failed && tid == 0) atomicCAS(p.status, 0, (int)TQ_ERR_TIMEOUT);
    cp_async_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (w == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(256) : "memory");
}

int observe_ctas(int head_dim) { return tq_sm_count() * (head_dim == 256 ? 1 : 2); }
int row_tiles_of(const tq_pages* g, int window, int Qh) { return (int)(((int64_t)window * (Qh / g->num_kv_heads) + OB_TILE - 1) / OB_TILE); }
size_t stats_bytes(const tq_pages* g, const tq_pages_batch* q, int window, int Qh) {
    return ((size_t)q->batch * g->num_kv_heads * row_tiles_of(g, window, Qh) + observe_ctas(g->head_dim)) * OB_TILE * sizeof(float2);
}
int observe_check(const tq_pages* g, const tq_pages_batch* q, int window, int Qh) {
    int rc = pages_check(g);
    if (rc == TQ_OK) rc = batch_check(g, q);
    if (rc != TQ_OK) return rc;
    if (window < 1 || Qh < 1 || Qh % g->num_kv_heads != 0) return TQ_ERR_SHAPE;
    if ((int64_t)window * (Qh / g->num_kv_heads) > (1 << 20)) return TQ_ERR_SHAPE;
    const int64_t lists = (int64_t)q->batch * g->num_kv_heads * row_tiles_of(g, window, Qh);
    if (lists * (((int64_t)q->max_seq_len + OB_TILE - 1) / OB_TILE) > MAX_UNITS) return TQ_ERR_SHAPE;
    return TQ_OK;
}
template <int D>
int launch(const ObserveParams& p, cudaStream_t st) {
    static TqSmemOptIn opt_a, opt_b;
    if (tq_opt_in_smem(tq_pages_observe_kernel<D, false>, observe_smem<D>(), opt_a) != TQ_OK ||
        tq_opt_in_smem(tq_pages_observe_kernel<D, true>, observe_smem<D>(), opt_b) != TQ_OK)
        return TQ_ERR_CUDA;
    const dim3 grid((unsigned)observe_ctas(D));
    const int rc = launch_behind(tq_pages_observe_kernel<D, false>, grid, OB_THREADS, observe_smem<D>(), st, p);
    return rc != TQ_OK ? rc : launch_behind(tq_pages_observe_kernel<D, true>, grid, OB_THREADS, observe_smem<D>(), st, p);
}

}  // namespace

extern "C" int tq_pages_observe_scratch_bytes(const tq_pages* pages, const tq_pages_batch* batch, int32_t window, int32_t num_q_heads,
                                              size_t* out) {
    if (!out) return TQ_ERR_NULL;
    const int rc = observe_check(pages, batch, window, num_q_heads);
    if (rc != TQ_OK) return rc;
    *out = stats_bytes(pages, batch, window, num_q_heads);
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
    if (scratch_bytes < stats_bytes(pages, batch, window, num_q_heads)) return TQ_ERR_WORKSPACE;
    ObserveParams p;
    p.g = pages_of(pages);
    p.q = batch_of(batch);
    p.query = static_cast<const uint8_t*>(query);
    p.Qh = num_q_heads;
    p.by_group = divisor(num_q_heads / pages->num_kv_heads);
    p.window = window;
    p.R = window * p.by_group.d;
    p.row_tiles = row_tiles_of(pages, window, num_q_heads);
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
