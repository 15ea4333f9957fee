// Attention of one new token per sequence over the exact paged cache.
//
// For a kv head with its group of G query heads:  s_gt = scale <q_g, k_t>,  out_g = sum_t 2^(s'_gt - m) v_t / sum_t 2^(s'_gt - m)
// with s' = s log2(e) and m a running maximum; keys and values are read once for every sixteen query heads of a kv head.  The bound
// is HBM: 4 D bytes a token and kv head against 4 G D operations.
//
// The batch is one list of UNITS (16 tokens of one kv head of one sequence) in the order sequence, head, token.  Every CTA
// (one per SM) takes an equal share of the list and every warp an equal share of that, whatever the lengths are: a share may
// begin and end inside a sequence.  A warp streams its units through a private ring of shared-memory stages (16-byte
// asynchronous copies, no barrier in the loop; a unit's keys and its values are a stage each, so that the wide heads have room
// for eight warps) and keeps an online softmax of its own.  (One bulk copy a row needs fewer instructions and is as fast for
// rows of 512 bytes, but an SM starts one in some 17 cycles: 940 us in the place of 577 for 64 mixed sequences of 256-byte
// rows.)  A (sequence, head) that lies within one warp's share is written at once; one that spans warps is joined in the CTA,
// one that spans CTAs through at most two partial results a CTA and a ticket, in the order of the list: the same launch gives
// the same bits every time.
//
// Measured: 64 sequences of 1024 to 32768 tokens, 64 / 8 heads of 128, 3.9 GB: 574 us, 6.7 TB/s (call after call:
// part of it still lies in L2).  One sequence of 32768, 16 / 4 heads of 256, 134 MB: 39 us, of which 23 are streaming, 4 the way to
// the first keys (lengths, table, rows) and 10 the joins (in the CTA 2.5, ticket 1.5, across CTAs 5: chains of loads in code that
// runs once).  A single short sequence: 7 us.
//
// Products: S^T = K Q^T and O^T = V^T P^T as m16n8k16, tokens resp. channels in the 16 rows, eight query heads in the columns,
// so that a group of up to eight pads nothing else.  tcgen05 would want 128 rows of operands through shared memory for eight
// useful columns; the tensor pipe is not what bounds this.  P goes into the second product as two 16-bit numbers, value and
// rest: one alone would cost as much precision as the rounding of the output.  Two bf16 numbers leave 2^-18 of a weight.  Two
// fp16 numbers leave 2^-22 of it, but nothing below half of fp16's smallest step, 2^-25, while a value row of zeros under the
// largest weight (a sink) makes the small weights all of the output: so fp16 weights are multiplied by 2^15 before they are
// split, and the factor is taken off again with the division by the sum.  What is lost of a weight is then at most 2^-40 of the largest
// one of the warp's share: up to 32768 values of size one, no more than half of the smallest step of an fp16 output.
#include <algorithm>

#include "tq_pages.cuh"

using namespace tqpg;

namespace {

struct DecodeParams {
    Pages g;
    Batch q;
    const uint8_t* query;
    uint8_t* out;
    int Qh, G, RT;            // query heads, per kv head, row tiles a kv head
    float scale_log2;
    float* partials;          // [2 * CTAs] slots, then [CTAs][warps]
    int32_t* tickets;         // [CTAs], zero between launches
    int32_t* status;
    float* scores;            // ledger: [batch * Qh][score_stride] scaled scores in the log2 domain, or NULL
    int64_t score_stride;
    float* lse;               // ledger: [batch * Qh] log2 of the weights' sum
};

constexpr int MAX_CTAS = 160;      // a join has a list of pieces, one a CTA at most

template <int D, int NT>
struct Shape {
    // 128 KB of stages an SM, 192 KB at head_dim 256, where a stage is 8 KB: 64 mixed sequences of head_dim 128 take 577 us with 128,
    // 620 with 192 (more copies under way than memory serves in order), 587 with 96.
    static constexpr int NW = 8;                                                   // warps
    static constexpr int NST = D == 64 ? 8 : D == 128 ? 4 : 3;                     // stages of a warp: 16 rows of keys or of values
    static constexpr int STAGE = 16 * D * 2;
    static constexpr int MASKS = 8;                                                // units whose row masks are kept: more than are under way
    static constexpr int ACC4 = D / 16 * NT * 32;                                  // float4 of a partial result, in fragment order
    static constexpr int SLOT = ACC4 * 4 + NT * 16;                                // floats: the sums, then (m, m, l, l) of the columns
    static constexpr int THREADS = NW * 32;
    static constexpr size_t SMEM = (size_t)NW * NST * STAGE + MAX_CTAS * 4 * NT * 16 + 1024;
    static_assert(SLOT * 4 <= NST * STAGE && NST / 2 + 2 <= MASKS && NST >= 2, "a warp's partial result takes the place of its ring");
};

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// The factor on the weights that go into the second product, and so on its sums (the sums of the weights are without it).
template <bool BF16>
constexpr float LIFT = BF16 ? 1.f : 32768.f;
// 2^(m - ref) where both may be -inf (nothing seen yet)
__device__ __forceinline__ float weight(float m, float ref) { return m == -INFINITY ? 0.f : ex2(m - ref); }

// A place in the list of units.
struct Place {
    int b, h, rt, c;   // sequence, kv head, row tile of its query heads, chunk of 16 tokens
    int len, nch;      // of the sequence: tokens, chunks
};
__device__ __forceinline__ void advance(Place& p, const DecodeParams& d) {
    if (++p.c < p.nch) return;
    p.c = 0;
    if (++p.rt < d.RT) return;
    p.rt = 0;
    if (++p.h < d.g.H) return;
    p.h = 0;
    do {
        ++p.b;
        p.len = seq_len(d.q, p.b, d.status);
    } while (p.len == 0 && p.b + 1 < d.q.batch);      // a share ends with its last unit: there is one ahead
    p.nch = (p.len + 15) >> 4;
}

struct Event {         // a (sequence, head) that spans CTAs
    int valid, b, h, rt, first, nch;
};

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(Shape<D, NT>::THREADS, 1) tq_pages_decode_kernel(const DecodeParams p) {
    using S = Shape<D, NT>;
    constexpr int NW = S::NW, NST = S::NST, KS = D / 16, ROWB = D * 2, SPLIT = NT == 1 ? 4 : 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (tq_smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint16_t s_mask[NW][S::MASKS];
    __shared__ int s_sum[NW], s_b[NW], s_pre[NW], s_len[NW], s_info[NW];
    __shared__ Event s_event[2], s_run[NW];
    __shared__ int s_border[2];
    __shared__ int s_last[2];                             // pieces, where this CTA is the last to arrive
    __shared__ float* s_piece[NW];
    __shared__ const float4* s_list[MAX_CTAS];
    float4* s_ml = reinterpret_cast<float4*>(smem + (size_t)NW * NST * S::STAGE);      // of the pieces of a join: [piece][column pair]

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int VH = p.g.H * p.RT;

    // Nothing is read before the launches ahead have finished; the ones behind may begin after that.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the share of this CTA and of this warp
    auto length = [&](int b) { return b < p.q.batch ? seq_len(p.q, b, p.status) : 0; };
    auto scan = [&](int c, int& total) {                  // inclusive over the CTA
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
        for (int i = 0; i < NW; ++i) {
            if (i < w) before += s_sum[i];
            total += s_sum[i];
        }
        __syncthreads();
        return x + before;
    };
    if (tid < 2) s_event[tid].valid = 0;
    const int len0 = length(tid);                         // the first sequences' stay in registers
    int all = 0, total0 = 0, incl0 = 0;
    for (int b0 = 0; b0 < p.q.batch; b0 += S::THREADS) {
        const int b = b0 + tid, len = b0 == 0 ? len0 : length(b);
        int total;
        const int incl = scan((len + 15) >> 4, total);
        if (b0 == 0) total0 = total, incl0 = incl;
        all += total;
        uint32_t empty = __ballot_sync(0xffffffffu, b < p.q.batch && len == 0 && b % (int)gridDim.x == (int)blockIdx.x);
        for (; empty; empty &= empty - 1) {               // nothing to attend to: zeros
            uint4* o = reinterpret_cast<uint4*>(p.out + (int64_t)(b0 + w * 32 + __ffs(empty) - 1) * p.Qh * ROWB);
            for (int i = lane; i < p.Qh * D / 8; i += 32) o[i] = make_uint4(0, 0, 0, 0);
        }
    }
    // The border between two CTAs' shares moves to the nearer end of a (sequence, head) of at most `keep` units: what such a one
    // costs a single CTA more is less than joining its pieces across CTAs (one sequence of 100 tokens and 8 kv heads 6.9 us in
    // the place of 9.7, 64 of 50 to 300 13.2 in the place of 15.5; of 500 tokens 10.2 in the place of 9.3).
    const int T = all * VH;
    const int share = max((T + (int)gridDim.x - 1) / (int)gridDim.x, NW);
    const int keep = share < 32 ? 24 : 32;
    if (tid < 2) s_border[tid] = T;
    __syncthreads();
    for (int b0 = 0, carry = 0; b0 < p.q.batch; b0 += S::THREADS) {
        const int len = b0 == 0 ? len0 : length(b0 + tid), c = (len + 15) >> 4;
        int total = total0;
        const int incl = b0 == 0 ? incl0 : scan(c, total);
        const int from = (carry + incl - c) * VH, to = (carry + incl) * VH;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t x = (int64_t)(blockIdx.x + i) * share;
            if (x >= from && x < to) {
                const int in = (int)(x - from) % c;
                s_border[i] = c > keep ? (int)x : 2 * in < c ? (int)x - in : (int)x - in + c;
            }
        }
        carry += total;
    }
    __syncthreads();
    const int lo = s_border[0], n = s_border[1] - lo;
    if (n <= 0) return;
    auto share_of = [&](int i) { return lo + (int)(((int64_t)n * i + NW - 1) / NW); };     // the first warp always has units
    const int x0 = share_of(w), x1 = share_of(w + 1);
    for (int b0 = 0, carry = 0; b0 < p.q.batch; b0 += S::THREADS) {
        const int len = b0 == 0 ? len0 : length(b0 + tid), c = (len + 15) >> 4;
        int total = total0;
        const int incl = b0 == 0 ? incl0 : scan(c, total);
        const int from = (carry + incl - c) * VH, to = (carry + incl) * VH;
        if (to > lo && from < lo + n)
            for (int i = 0; i < NW; ++i) {
                const int x = share_of(i);
                if (x >= from && x < to) {
                    s_b[i] = b0 + tid;
                    s_pre[i] = from;
                    s_len[i] = len;
                }
            }
        carry += total;
    }
    __syncthreads();

    Place at = {}, ahead;
    int units = x1 - x0, first = 0;                       // first: where the current (sequence, head) begins in the list
    if (units > 0) {
        at.b = s_b[w];
        at.len = s_len[w];
        at.nch = (at.len + 15) >> 4;
        const int rel = x0 - s_pre[w], vh = rel / at.nch;
        at.c = rel - vh * at.nch;
        at.h = vh / p.RT;
        at.rt = vh - at.h * p.RT;
        first = x0 - at.c;
    }
    ahead = at;

    // ---- loading: stage i holds the keys (even) or values (odd) of unit i / 2, row by row
    uint8_t* ring = smem + (size_t)w * NST * S::STAGE;
    const uint32_t ring_u = tq_smem_u32(ring);
    const int my_row = lane & 15;
    int entry = 0;                                        // this lane's row of the unit ahead: its page ...
    int64_t row_off = 0;                                  // ... and its place in the planes
    auto look_up = [&]() {                                // asked for one unit before it is needed
        const int t = ahead.c * 16 + my_row;
        entry = t < ahead.len ? p.q.table[(int64_t)ahead.b * p.q.table_stride + p.g.by_page.quotient(t)] : -1;
    };
    int issued = 0, wr = 0;                               // stages asked for so far, place of the next
    uint32_t rows_there = 0;
    constexpr int LPR = D / 8, RPI = 32 / LPR;            // lanes a row, rows an instruction
    const int r0 = lane / LPR, byte = (lane % LPR) * 16;
    const bool whole = (p.g.page & 15) == 0;              // a unit lies in one page
    auto issue = [&]() {
        if (issued < 2 * units) {
            const bool values = issued & 1;
            if (!values) {
                const int t = ahead.c * 16 + my_row;
                const bool there = (uint32_t)entry < (uint64_t)p.g.num_blocks;
                if (!there && t < ahead.len) atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
                row_off = (int64_t)entry * p.g.sb + (int64_t)(t - p.g.by_page.quotient(t) * p.g.page) * p.g.st + ahead.h * p.g.sh;
                rows_there = __ballot_sync(0xffffffffu, there) & 0xffffu;
                if (lane == 0) s_mask[w][(issued >> 1) % S::MASKS] = (uint16_t)rows_there;
                if (issued + 2 < 2 * units) {
                    advance(ahead, p);
                    look_up();
                }
            }
            const uint8_t* plane = (values ? p.g.v : p.g.k) + byte;
            // 16-byte piece c of row r lies at piece c ^ (r % 8): eight rows of one piece are in different banks
            const uint32_t dst = ring_u + wr * S::STAGE + r0 * ROWB + (byte ^ (r0 << 4));
            if (whole && rows_there == 0xffffu) {
                const uint8_t* src = plane + __shfl_sync(0xffffffffu, row_off, 0) + r0 * p.g.st;
#pragma unroll
                for (int i = 0; i < 16 / RPI; ++i) cp_async16((dst ^ (((i * RPI) & 7) << 4)) + i * RPI * ROWB, src + i * RPI * p.g.st, true);
            } else {                                      // absent rows become zeros: times a weight of zero they must not be NaN
#pragma unroll
                for (int i = 0; i < 16 / RPI; ++i) {
                    const int64_t off = __shfl_sync(0xffffffffu, row_off, i * RPI + r0);
                    const bool there = (rows_there >> (i * RPI + r0)) & 1;
                    cp_async16((dst ^ (((i * RPI) & 7) << 4)) + i * RPI * ROWB, plane + (there ? off : 0), there);
                }
            }
            ++issued;
            wr = wr + 1 == NST ? 0 : wr + 1;
        }
        cp_async_commit();
    };
    int rd = 0;                                           // the stage that is read next
    auto arrived = [&]() {
        cp_async_wait<NST - 1>();
        __syncwarp();
        return ring_u + rd * S::STAGE;
    };
    auto release = [&]() {
        __syncwarp();
        rd = rd + 1 == NST ? 0 : rd + 1;
        issue();
    };
    // ---- the current (sequence, head)
    uint32_t qf[NT][KS][2];
    float acc[KS][NT][4], m[NT][2], l[NT][2];
    auto rows_of = [&](int rt) { return min(p.G - rt * 8 * NT, 8 * NT); };                // query heads of a row tile
    auto first_row = [&](int b, int h, int rt) { return (int64_t)b * p.Qh + h * p.G + rt * 8 * NT; };
    float* sc = nullptr;                                  // ledger: where this lane's scores of the current unit go
    auto begin = [&]() {
        const int rows = rows_of(at.rt);
        if (p.scores != nullptr) sc = p.scores + (first_row(at.b, at.h, at.rt) + 2 * t4) * p.score_stride + at.c * 16 + g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint8_t* q = p.query + (first_row(at.b, at.h, at.rt) + nt * 8 + g) * ROWB + t4 * 4;
            const bool there = nt * 8 + g < rows;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[nt][ks][0] = there ? *reinterpret_cast<const uint32_t*>(q + ks * 32) : 0u;
                qf[nt][ks][1] = there ? *reinterpret_cast<const uint32_t*>(q + ks * 32 + 16) : 0u;
            }
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int ct = 0; ct < KS; ++ct)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[ct][nt][i] = 0.f;
        }
    };
    auto sum_l = [&]() {                                  // the lanes' shares of the columns' sums
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], o);
    };
    auto write_out = [&](int b, int h, int rt) {          // l summed
        const int rows = rows_of(rt);
        const int64_t row0 = first_row(b, h, rt);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float i0 = l[nt][0] == 0.f ? 0.f : 1.f / LIFT<BF16> / l[nt][0], i1 = l[nt][1] == 0.f ? 0.f : 1.f / LIFT<BF16> / l[nt][1];
            uint8_t* o = p.out + (row0 + nt * 8 + g) * ROWB + t4 * 4;
#pragma unroll
            for (int ct = 0; ct < KS; ++ct) {
                const uint32_t a = transpose8(pack<BF16>(acc[ct][nt][0] * i0, acc[ct][nt][1] * i1));
                const uint32_t c = transpose8(pack<BF16>(acc[ct][nt][2] * i0, acc[ct][nt][3] * i1));
                if (nt * 8 + g < rows) {
                    *reinterpret_cast<uint32_t*>(o + ct * 32) = a;
                    *reinterpret_cast<uint32_t*>(o + ct * 32 + 16) = c;
                }
            }
            if (p.lse != nullptr && g == 0)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (nt * 8 + 2 * t4 + j < rows)
                        p.lse[row0 + nt * 8 + 2 * t4 + j] = l[nt][j] == 0.f ? INFINITY : m[nt][j] + log2f(l[nt][j]);
        }
    };
    // A piece's sums as they lie in the lanes, then (m, m, l, l) of every pair of columns.  Columns without a query head are
    // neither written nor read.
    auto write_slot = [&](float* slot) {                  // l summed
        const int rows = rows_of(at.rt);
        float4* s = reinterpret_cast<float4*>(slot);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt * 8 + 2 * t4 >= rows) continue;
#pragma unroll
            for (int ct = 0; ct < KS; ++ct)
                s[(ct * NT + nt) * 32 + lane] = make_float4(acc[ct][nt][0], acc[ct][nt][1], acc[ct][nt][2], acc[ct][nt][3]);
            if (g == 0) s[S::ACC4 + nt * 4 + t4] = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
        }
    };
    auto add_slot = [&](const float* slot) {
        const int rows = rows_of(at.rt);
        const float4* s = reinterpret_cast<const float4*>(slot);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt * 8 + 2 * t4 >= rows) continue;
            const float4 ml = s[S::ACC4 + nt * 4 + t4];
            const float m0 = fmaxf(m[nt][0], ml.x), m1 = fmaxf(m[nt][1], ml.y);
            const float a0 = weight(m[nt][0], m0), a1 = weight(m[nt][1], m1), b0 = weight(ml.x, m0), b1 = weight(ml.y, m1);
            l[nt][0] = l[nt][0] * a0 + ml.z * b0;
            l[nt][1] = l[nt][1] * a1 + ml.w * b1;
            m[nt][0] = m0;
            m[nt][1] = m1;
#pragma unroll
            for (int ct = 0; ct < KS; ++ct) {
                const float4 v = s[(ct * NT + nt) * 32 + lane];
                acc[ct][nt][0] = acc[ct][nt][0] * a0 + v.x * b0;
                acc[ct][nt][1] = acc[ct][nt][1] * a1 + v.y * b1;
                acc[ct][nt][2] = acc[ct][nt][2] * a0 + v.z * b0;
                acc[ct][nt][3] = acc[ct][nt][3] * a1 + v.w * b1;
            }
        }
    };
    auto global_slot = [&](int cta, int which) { return p.partials + ((int64_t)cta * 2 + which) * S::SLOT; };
    // a warp's piece of a (sequence, head) that an earlier warp began: in place of its ring, or in memory while that is in use
    auto own_slot = [&](int i) { return reinterpret_cast<float*>(smem + (size_t)i * NST * S::STAGE); };
    auto warp_slot = [&](int i) { return p.partials + ((int64_t)gridDim.x * 2 + blockIdx.x * NW + i) * S::SLOT; };
    float* head_piece = nullptr;

    // flags: 0 no units; 1 this warp's first piece ends a (sequence, head) that an earlier warp began; 2 its whole share is such a
    // piece and goes on; 3 begins with a (sequence, head) of its own
    int flag = 0;
    bool open = false;          // the last piece goes on behind this warp's share
    if (units > 0) {
        look_up();
        flag = at.c == 0 ? 3 : (at.nch - at.c <= units ? 1 : 2);
        begin();
    }
    // the query has been asked for: the first keys come behind it
#pragma unroll 1
    for (int i = 0; i < NST; ++i) issue();

    // ldmatrix: this lane's row and 16-byte piece of a 16 x 16 tile of the keys, and of the values (transposed)
    const uint32_t k_at = (((lane >> 3) & 1) * 8 + (lane & 7)) * ROWB + (((lane >> 4) ^ (lane & 7)) << 4);
    const uint32_t v_at = ((lane >> 4) * 8 + (lane & 7)) * ROWB + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
#pragma unroll 1
    for (int u = 0; u < units; ++u) {
        const uint32_t kb = arrived();
        const uint32_t mask = s_mask[w][u % S::MASKS];
        float s[NT][4], part[NT][SPLIT][4];               // several chains of products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4 * SPLIT; ++i) part[nt][i >> 2][i & 3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t a[4];
            ldsm4(a, (kb + k_at) ^ (ks * 32));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<BF16>(part[nt][ks % SPLIT], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
        release();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[nt][i] = part[nt][0][i] + part[nt][1][i];
                if (SPLIT == 4) s[nt][i] += part[nt][SPLIT - 2][i] + part[nt][SPLIT - 1][i];
                s[nt][i] *= p.scale_log2;
            }
        if (mask != 0xffffu) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!((mask >> (g + (i >> 1) * 8)) & 1)) s[nt][i] = -INFINITY;
        }
        if (p.scores != nullptr) {
            const int rows = rows_of(at.rt);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (nt * 8 + 2 * t4 + (i & 1) < rows) sc[(nt * 8 + (i & 1)) * p.score_stride + (i >> 1) * 8] = s[nt][i];
            sc += 16;
        }
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            grows |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] || fmaxf(s[nt][1], s[nt][3]) > m[nt][1];
        if (__any_sync(0xffffffffu, grows)) {             // a score above the running maximum
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float mx = fmaxf(m[nt][j], fmaxf(s[nt][j], s[nt][j + 2]));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float a = weight(m[nt][j], mx);
                    m[nt][j] = mx;
                    l[nt][j] *= a;
#pragma unroll
                    for (int ct = 0; ct < KS; ++ct) {
                        acc[ct][nt][j] *= a;
                        acc[ct][nt][j + 2] *= a;
                    }
                }
        }
        uint32_t hi[NT][2], rest[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float r0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], r1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float a = ex2(s[nt][2 * k] - r0), c = ex2(s[nt][2 * k + 1] - r1);
                l[nt][0] += a;
                l[nt][1] += c;
                a *= LIFT<BF16>;
                c *= LIFT<BF16>;
                const uint32_t h = pack<BF16>(a, c);
                const float2 back = unpack<BF16>(h);
                hi[nt][k] = transpose8(h);
                rest[nt][k] = transpose8(pack<BF16>(a - back.x, c - back.y));
            }
        }
        const uint32_t vb = arrived();
#pragma unroll
        for (int c4 = 0; c4 < KS; c4 += 4) {              // four tiles at a time: no product waits for the one before it
            uint32_t a[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ldsm4t(a[i], (vb + v_at) ^ ((c4 + i) * 32));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<BF16>(acc[c4 + i][nt], a[i], hi[nt][0], hi[nt][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<BF16>(acc[c4 + i][nt], a[i], rest[nt][0], rest[nt][1]);
            }
        }

        release();

        const bool ends = at.c + 1 == at.nch;
        const bool last_unit = u + 1 == units;
        if (ends || last_unit) {
            sum_l();
            if (ends && first >= x0) {
                write_out(at.b, at.h, at.rt);
            } else {
                open = !ends;
                // a piece of an earlier warp's (sequence, head) that ends in the first warp began in an earlier CTA
                const bool to_event = ends && w == 0;
                if (to_event) {
                    if (lane == 0) s_event[0] = Event{1, at.b, at.h, at.rt, first, at.nch};
                }
                float* slot = to_event ? global_slot(blockIdx.x, 0) : last_unit ? own_slot(w) : warp_slot(w);     // the ring is in use up to the last unit
                if (first < x0) head_piece = slot;
                write_slot(slot);
            }
        }
        if (!last_unit) {
            advance(at, p);
            if (ends) {
                first = x0 + u + 1;
                begin();
            }
        }
    }
    cp_async_wait<0>();

    // ---- joins.  A RUN is a (sequence, head) whose first piece in this CTA is a warp's last one and goes on in the warps behind it.
    // Several runs: each warp adds up its own in its registers.  One run, as in a long sequence: all threads work on it.  A run
    // that does not hold all of its (sequence, head) becomes a partial result of the CTA, and the CTA that arrives last adds up
    // all of those, in the order of the list.
    const bool owner = open && !(flag == 2 && w > 0);
    if (lane == 0) {
        s_info[w] = flag | (owner ? 4 : 0);
        s_piece[w] = head_piece;
        if (owner) s_run[w] = Event{1, at.b, at.h, at.rt, first, at.nch};
    }
    __syncthreads();
    const int info = lane < NW ? s_info[lane] : 0;
    const uint32_t filled = __ballot_sync(0xffffffffu, (info & 3) != 0), closing = __ballot_sync(0xffffffffu, (info & 3) == 1),
                   owners = __ballot_sync(0xffffffffu, (info & 4) != 0);
    // the warps whose first pieces follow that of warp i, and whether the last of them ends the (sequence, head)
    auto followers = [&](int i, bool& done) {
        uint32_t behind = filled & ~((2u << i) - 1u);
        const uint32_t end = closing & behind;
        done = end != 0u;
        if (done) behind &= ((end & (0u - end)) << 1) - 1u;
        return behind;
    };
    const bool together = __popc(owners) == 1;
    if (owner && !together) {
        bool done;
        for (uint32_t more = followers(w, done); more; more &= more - 1) add_slot(s_piece[__ffs(more) - 1]);
        if (done && first >= lo) {
            write_out(at.b, at.h, at.rt);
        } else {
            const int which = first >= lo ? 1 : 0;
            write_slot(global_slot(blockIdx.x, which));
            if (lane == 0) s_event[which] = s_run[w];
        }
    }
#pragma unroll 1
    for (int round = together ? 0 : 1; round < 3; ++round) {      // the CTA's one run, then the two (sequence, head)s it may be the last to join
        Event ev;
        int pieces;
        float4* to = nullptr;                             // partial result, or NULL: the output
        if (round == 0) {
            const int i = __ffs(owners) - 1;
            bool done;
            const uint32_t more = followers(i, done);
            ev = s_run[i];
            pieces = 1 + __popc(more);
            const int which = ev.first >= lo ? 1 : 0;
            if (!(done && which == 1)) to = reinterpret_cast<float4*>(global_slot(blockIdx.x, which));
            if (tid == 0 && to != nullptr) s_event[which] = ev;
            if (tid == i) s_list[0] = reinterpret_cast<const float4*>(own_slot(i));
            if (tid < NW && ((more >> tid) & 1)) s_list[1 + __popc(more & ((1u << tid) - 1u))] = reinterpret_cast<const float4*>(s_piece[tid]);
        } else {
            if (round == 1) {
                __syncthreads();
                if (!s_event[0].valid && !s_event[1].valid) return;
                if (tid < 2) {
                    s_last[tid] = 0;
                    if (s_event[tid].valid) {
                        const int from = s_event[tid].first / share, to = (s_event[tid].first + s_event[tid].nch - 1) / share;
                        int before;                       // releases this CTA's pieces, acquires the others'
                        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.tickets + from) : "memory");
                        if (before == to - from) {
                            p.tickets[from] = 0;          // for the next launch
                            s_last[tid] = to - from + 1;
                        }
                    }
                }
            }
            __syncthreads();
            pieces = s_last[round - 1];
            if (pieces == 0) continue;
            ev = s_event[round - 1];
            const int from = ev.first / share;
            if (tid < pieces) s_list[tid] = reinterpret_cast<const float4*>(global_slot(from + tid, tid == 0 ? 1 : 0));
        }
        __syncthreads();
        const int rows = rows_of(ev.rt), lp = NT == 2 || rows > 4 ? 2 : rows > 2 ? 1 : 0;    // log2 of the column pairs that count
        const int64_t row0 = first_row(ev.b, ev.h, ev.rt);
#pragma unroll 1
        for (int base = 0; base < (KS * NT * 8) << lp; base += S::THREADS) {
            constexpr int STEP = 20;                      // a long sequence's 37 pieces in two rounds of loads
            const int i = base + tid, t = i & ((1 << lp) - 1), gg = (i >> lp) & 7, tile = i >> (lp + 3), nt = tile % NT, ct = tile / NT;
            const int row = nt * 8 + 2 * t, f = tile * 32 + gg * 4 + t;
            const bool there = row < rows && tile < KS * NT;
            float4 v[STEP], a = make_float4(0.f, 0.f, 0.f, 0.f);
            auto ask = [&](int k0) {
#pragma unroll
                for (int k = 0; k < STEP; ++k)
                    if (there && k0 + k < pieces) v[k] = s_list[k0 + k][f];
            };
            ask(0);
            if (base == 0) {                              // maxima and sums of all pieces
                for (int j = tid; j < pieces * 4 * NT; j += S::THREADS)
                    if (2 * (j % (4 * NT)) < rows) s_ml[j] = s_list[j / (4 * NT)][S::ACC4 + j % (4 * NT)];
                __syncthreads();
            }
            if (!there) continue;
            const float4* ml = s_ml + nt * 4 + t;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll 4
            for (int k = 0; k < pieces; ++k) {
                const float4 x = ml[k * 4 * NT];
                m0 = fmaxf(m0, x.x);
                m1 = fmaxf(m1, x.y);
            }
#pragma unroll 1
            for (int k0 = 0; k0 < pieces; k0 += STEP) {
                if (k0 > 0) ask(k0);
#pragma unroll
                for (int k = 0; k < STEP; ++k) {
                    if (k0 + k >= pieces) break;
                    const float4 x = ml[(k0 + k) * 4 * NT];
                    const float w0 = weight(x.x, m0), w1 = weight(x.y, m1);
                    l0 = fmaf(x.z, w0, l0);
                    l1 = fmaf(x.w, w1, l1);
                    a.x = fmaf(v[k].x, w0, a.x);
                    a.y = fmaf(v[k].y, w1, a.y);
                    a.z = fmaf(v[k].z, w0, a.z);
                    a.w = fmaf(v[k].w, w1, a.w);
                }
            }
            if (to != nullptr) {
                to[f] = a;
                if (ct == 0 && gg == 0) to[S::ACC4 + nt * 4 + t] = make_float4(m0, m1, l0, l1);
                continue;
            }
            using E = TqElem<BF16 ? TQ_BF16 : TQ_F16>;
            const int64_t o = (row0 + row) * D + ct * 16 + gg;
            const float i0 = l0 == 0.f ? 0.f : 1.f / LIFT<BF16> / l0, i1 = l1 == 0.f ? 0.f : 1.f / LIFT<BF16> / l1;
            E::store(p.out, o, a.x * i0);
            E::store(p.out, o + 8, a.z * i0);
            if (row + 1 < rows) {
                E::store(p.out, o + D, a.y * i1);
                E::store(p.out, o + D + 8, a.w * i1);
            }
            if (p.lse != nullptr && ct == 0 && gg == 0) {
                p.lse[row0 + row] = l0 == 0.f ? INFINITY : m0 + log2f(l0);
                if (row + 1 < rows) p.lse[row0 + row + 1] = l1 == 0.f ? INFINITY : m1 + log2f(l1);
            }
        }
    }
}

// mass[b][h][t] += sum over the group's heads of 2^(score - lse): 4 G bytes read and 8 moved a token and head, against the 4 D
// that the attention reads.  16 sequences of 4001 to 8192, 32 / 8 heads of 128: 7 us behind the attention's 73.
constexpr int LEDGER_TOK = 4;      // tokens a thread
__global__ void __launch_bounds__(256) tq_pages_ledger_kernel(const Batch q, const float* scores, int64_t score_stride,
                                                              const float* lse, int H, int G, float* mass, int64_t mass_stride,
                                                              int32_t* status) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.x / H;
    const int n = seq_len(q, b, status);
    const int64_t row = (int64_t)blockIdx.x * G;
    float* to = mass + blockIdx.x * mass_stride;
    for (int tile = blockIdx.y * 256 * LEDGER_TOK; tile < n; tile += gridDim.y * 256 * LEDGER_TOK) {
        const int t0 = tile + threadIdx.x;
        float sum[LEDGER_TOK], old[LEDGER_TOK];
#pragma unroll
        for (int k = 0; k < LEDGER_TOK; ++k) {
            sum[k] = 0.f;
            if (t0 + k * 256 < n) old[k] = to[t0 + k * 256];
        }
#pragma unroll 4
        for (int i = 0; i < G; ++i) {
            const float* s = scores + (row + i) * score_stride + t0;
            const float base = lse[row + i];
#pragma unroll
            for (int k = 0; k < LEDGER_TOK; ++k)
                if (t0 + k * 256 < n) sum[k] += ex2(__ldcs(s + k * 256) - base);
        }
#pragma unroll
        for (int k = 0; k < LEDGER_TOK; ++k)
            if (t0 + k * 256 < n) to[t0 + k * 256] = old[k] + sum[k];
    }
}

// The scores of a ledger's call take 4 bytes a query head and token of the host's bound, whatever the lengths are.  Beyond
// SCORES_MOST the batch goes through in slices of sequences, one at least, over the same scratch memory: 256 sequences of 300 to
// 600 tokens, 64 query heads, under a bound of 131072 take 0.5 GB in the place of 8.6 and 365 us in 17 slices; 64 of them 90 us in
// five.
constexpr size_t SCORES_MOST = (size_t)512 << 20;
struct Scratch {
    size_t partials, lse, scores, bytes;
    int64_t score_stride;
    int slice;                // sequences at a time
};
int row_tiles(int G) { return (G + 15) / 16; }
Scratch scratch_of(const tq_pages* g, const tq_pages_batch* q, int Qh, bool ledger) {
    const int nt = Qh / g->num_kv_heads > 8 ? 2 : 1;
    const size_t slot = (size_t)g->head_dim / 16 * nt * 128 + nt * 16;      // Shape<>::SLOT, Shape<>::NW warps
    Scratch s;
    s.score_stride = ((int64_t)q->max_seq_len + 15) / 16 * 16;
    const size_t each = (size_t)Qh * s.score_stride * 4;
    s.slice = !ledger || each * q->batch <= SCORES_MOST ? q->batch : each >= SCORES_MOST ? 1 : (int)(SCORES_MOST / each);
    s.partials = 0;
    s.lse = (size_t)tq_sm_count() * (2 + 8) * slot * 4;
    s.scores = s.lse + (ledger ? ((size_t)s.slice * Qh * 4 + 255) / 256 * 256 : 0);
    s.bytes = s.scores + (ledger ? s.slice * each : 0);
    return s;
}

template <int D, int NT, bool BF16>
int launch(const DecodeParams& p, int ctas, cudaStream_t st) {
    using S = Shape<D, NT>;
    static TqSmemOptIn opt_in;
    if (tq_opt_in_smem(tq_pages_decode_kernel<D, NT, BF16>, S::SMEM, opt_in) != TQ_OK) return TQ_ERR_CUDA;
    return launch_behind(tq_pages_decode_kernel<D, NT, BF16>, dim3((unsigned)ctas), S::THREADS, S::SMEM, st, p);
}
template <int D, int NT>
int launch_dtype(const DecodeParams& p, int dtype, int ctas, cudaStream_t st) {
    return dtype == TQ_BF16 ? launch<D, NT, true>(p, ctas, st) : launch<D, NT, false>(p, ctas, st);
}

int decode_check(const tq_pages* g, const tq_pages_batch* q, int32_t num_q_heads) {
    int rc = pages_check(g);
    if (rc == TQ_OK) rc = batch_check(g, q);
    if (rc != TQ_OK) return rc;
    if (num_q_heads < 1 || num_q_heads % g->num_kv_heads != 0) return TQ_ERR_SHAPE;
    const int64_t heads = (int64_t)g->num_kv_heads * row_tiles(num_q_heads / g->num_kv_heads);
    if (heads * q->batch * (((int64_t)q->max_seq_len + 15) / 16) > MAX_UNITS) return TQ_ERR_SHAPE;
    return TQ_OK;
}

}  // namespace

extern "C" size_t tq_pages_ticket_bytes(void) { return (size_t)tq_sm_count() * sizeof(int32_t); }

extern "C" int tq_pages_decode_scratch_bytes(const tq_pages* pages, const tq_pages_batch* batch, int32_t num_q_heads, int32_t with_mass,
                                             size_t* out) {
    if (!out) return TQ_ERR_NULL;
    const int rc = decode_check(pages, batch, num_q_heads);
    if (rc != TQ_OK) return rc;
    *out = scratch_of(pages, batch, num_q_heads, with_mass != 0).bytes;
    return TQ_OK;
}

extern "C" int tq_pages_decode(const tq_pages* pages, const tq_pages_batch* batch, const void* query, int32_t num_q_heads, float scale,
                               void* out, float* mass, int64_t mass_stride, void* scratch, size_t scratch_bytes, int32_t* tickets,
                               int32_t* status, void* stream) {
    int rc = decode_check(pages, batch, num_q_heads);
    if (rc != TQ_OK) return rc;
    if (!query || !out || !scratch || !tickets || !status) return TQ_ERR_NULL;
    if (((uintptr_t)query & 15) || ((uintptr_t)out & 15) || ((uintptr_t)scratch & 15)) return TQ_ERR_ALIGN;
    if (mass && mass_stride < batch->max_seq_len) return TQ_ERR_RANGE;
    const Scratch s = scratch_of(pages, batch, num_q_heads, mass != nullptr);
    if (scratch_bytes < s.bytes) return TQ_ERR_WORKSPACE;
    DecodeParams p;
    p.g = pages_of(pages);
    p.q = batch_of(batch);
    p.query = static_cast<const uint8_t*>(query);
    p.out = static_cast<uint8_t*>(out);
    p.Qh = num_q_heads;
    p.G = num_q_heads / pages->num_kv_heads;
    p.RT = row_tiles(p.G);
    p.scale_log2 = scale * 1.4426950408889634f;
    uint8_t* base = static_cast<uint8_t*>(scratch);
    p.partials = reinterpret_cast<float*>(base + s.partials);
    p.tickets = tickets;
    p.status = status;
    p.scores = mass ? reinterpret_cast<float*>(base + s.scores) : nullptr;
    p.score_stride = s.score_stride;
    p.lse = mass ? reinterpret_cast<float*>(base + s.lse) : nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    const int sms = tq_sm_count(), ctas = sms < MAX_CTAS ? sms : MAX_CTAS, two = p.G > 8;
    tq_note_launch(st, TQ_LAUNCH_WAITED);
    const int tile = 256 * LEDGER_TOK;
    const int64_t rows = (int64_t)s.slice * num_q_heads * pages->head_dim * 2;      // bytes of a slice's queries and outputs
    for (int b = 0; b < batch->batch; b += s.slice) {
        p.q.batch = batch->batch - b < s.slice ? batch->batch - b : s.slice;
        switch (pages->head_dim) {
            case 64: rc = two ? launch_dtype<64, 2>(p, pages->dtype, ctas, st) : launch_dtype<64, 1>(p, pages->dtype, ctas, st); break;
            case 128: rc = two ? launch_dtype<128, 2>(p, pages->dtype, ctas, st) : launch_dtype<128, 1>(p, pages->dtype, ctas, st); break;
            default: rc = two ? launch_dtype<256, 2>(p, pages->dtype, ctas, st) : launch_dtype<256, 1>(p, pages->dtype, ctas, st); break;
        }
        if (rc != TQ_OK || !mass) return rc;
        // four waves of CTAs, not one for every tile that the bound allows: 512 rows under a bound of 131072 tokens are 65536 of those
        const int64_t heads = (int64_t)p.q.batch * pages->num_kv_heads, tiles = ((int64_t)batch->max_seq_len + tile - 1) / tile;
        const int64_t most = std::max<int64_t>(1, 4 * 8 * sms / heads);
        const dim3 grid((unsigned)heads, (unsigned)std::min(tiles, most));
        rc = launch_behind(tq_pages_ledger_kernel, grid, 256, 0, st, p.q, (const float*)p.scores, p.score_stride, (const float*)p.lse,
                           (int)pages->num_kv_heads, p.G, mass, mass_stride, status);
        if (rc != TQ_OK) return rc;
        p.q.table += (int64_t)s.slice * p.q.table_stride;
        p.q.lens += s.slice;
        p.query += rows;
        p.out += rows;
        mass += (int64_t)s.slice * pages->num_kv_heads * mass_stride;
    }
    return TQ_OK;
}
