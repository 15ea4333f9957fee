// Attention of one new token per sequence over the exact paged cache.
//
// For a kv head with its group of G query heads:  s_gt = scale <q_g, k_t>,  out_g = sum_t 2^(s'_gt - m) v_t / sum_t 2^(s'_gt - m)
// with s' = s log2(e) and m a running maximum; keys and values are read once.  The bound is HBM: 4 D bytes a token and kv head
// against 4 G D operations.
//
// The batch is one list of UNITS (16 tokens of one kv head of one sequence) in the order sequence, head, token.  Every CTA
// (one per SM) takes an equal share of the list and every warp an equal share of that, whatever the lengths are: a share may
// begin and end inside a sequence.  A warp streams its units through a private ring of shared-memory stages (16-byte
// asynchronous copies, no barrier in the loop) and keeps an online softmax of its own.  A (sequence, head) that lies within
// one warp's share is written at once; one that spans warps is joined in shared memory, one that spans CTAs through at most
// two partial results a CTA and a ticket, in the order of the list: the same launch gives the same bits every time.
//
// Products: S^T = K Q^T and O^T = V^T P^T as m16n8k16, tokens resp. channels in the 16 rows, eight query heads in the columns,
// so that a group of up to eight pads nothing else.  tcgen05 would want 128 rows of operands through shared memory for eight
// useful columns; the tensor pipe is not what bounds this.  P goes into the second product as two 16-bit numbers (value and
// rest, 2^-16 relative): one alone would cost as much precision as the rounding of the output.
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
    float* partials;          // [2 * CTAs] slots
    int32_t* tickets;         // [CTAs], zero between launches
    int32_t* status;
    float* scores;            // ledger: [batch * Qh][score_stride] scaled scores in the log2 domain, or NULL
    int64_t score_stride;
    float* lse;               // ledger: [batch * Qh] log2 of the weights' sum
};

template <int D, int NT>
struct Shape {
    static constexpr int NW = NT == 1 ? (D == 256 ? 4 : 8) : (D == 256 ? 3 : 6);   // warps
    static constexpr int NST = D == 64 ? 6 : 3;                                    // stages of a warp
    static constexpr int UNIT = 16 * D * 2 * 2;                                    // bytes of a unit, keys then values
    static constexpr int ACC4 = D / 16 * NT * 32;                                  // float4 of a partial result, in fragment order
    static constexpr int SLOT = ACC4 * 4 + NT * 16;                                // floats: the sums, then (m, m, l, l) of the columns
    static constexpr int THREADS = NW * 32;
    static constexpr size_t SMEM = (size_t)NW * NST * UNIT + (size_t)NW * SLOT * 4;
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
// 2^(m - ref) where both may be -inf (nothing seen yet)
__device__ __forceinline__ float weight(float m, float ref) { return m == -INFINITY ? 0.f : ex2(m - ref); }

// A place in the list of units.
struct Place {
    int b, vh, c;      // sequence, virtual head (kv head * row tiles + row tile), chunk of 16 tokens
    int len, nch;      // of the sequence: tokens, chunks
};
__device__ __forceinline__ void advance(Place& p, const DecodeParams& d, int VH) {
    if (++p.c < p.nch) return;
    p.c = 0;
    if (++p.vh < VH) return;
    p.vh = 0;
    do {
        ++p.b;
        p.len = seq_len(d.q, p.b, d.status);
    } while (p.len == 0 && p.b + 1 < d.q.batch);      // a share ends with its last unit: there is one ahead
    p.nch = (p.len + 15) >> 4;
}

struct Event {         // a (sequence, head) that spans CTAs
    int valid, b, vh, first, nch;
};

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(Shape<D, NT>::THREADS, 1) tq_pages_decode_kernel(const DecodeParams p) {
    using S = Shape<D, NT>;
    constexpr int NW = S::NW, NST = S::NST, KS = D / 16, ROWB = D * 2;
    constexpr int LPR = D / 8, RPI = 32 / LPR;            // lanes a row, rows an instruction
    extern __shared__ __align__(128) uint8_t smem[];
    float* slots = reinterpret_cast<float*>(smem + (size_t)NW * NST * S::UNIT);
    __shared__ uint32_t s_mask[NW][NST];
    __shared__ int s_sum[NW], s_b[NW], s_pre[NW], s_flag[NW];
    __shared__ Event s_event[2];
    __shared__ int s_last[2];
    __shared__ float s_inv[16];

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int VH = p.g.H * p.RT;

    // ---- the share of this CTA and of this warp
    auto chunks = [&](int b) { return b < p.q.batch ? (seq_len(p.q, b, p.status) + 15) >> 4 : 0; };
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
    int all = 0;
    for (int b0 = 0; b0 < p.q.batch; b0 += S::THREADS) {
        int total;
        scan(chunks(b0 + tid), total);
        all += total;
    }
    const int T = all * VH;
    for (int b = blockIdx.x * NW + w; b < p.q.batch; b += gridDim.x * NW)      // nothing to attend to: zeros
        if (seq_len(p.q, b, p.status) == 0)
            for (int i = lane; i < p.Qh * D / 8; i += 32)
                reinterpret_cast<uint4*>(p.out + (int64_t)b * p.Qh * ROWB)[i] = make_uint4(0, 0, 0, 0);
    const int share = max((T + (int)gridDim.x - 1) / (int)gridDim.x, NW);
    const int lo = min((int64_t)T, (int64_t)blockIdx.x * share), n = min(T - lo, share);
    if (n <= 0) return;
    auto share_of = [&](int i) { return lo + (int)(((int64_t)n * i + NW - 1) / NW); };     // the first warp always has units
    const int x0 = share_of(w), x1 = share_of(w + 1);
    if (tid < 2) s_event[tid].valid = 0;
    {
        int carry = 0;
        for (int b0 = 0; b0 < p.q.batch; b0 += S::THREADS) {
            int total;
            const int c = chunks(b0 + tid), incl = scan(c, total);
            const int from = (carry + incl - c) * VH, to = (carry + incl) * VH;
            for (int i = 0; i < NW; ++i) {
                const int x = share_of(i);
                if (x >= from && x < to) {
                    s_b[i] = b0 + tid;
                    s_pre[i] = from;
                }
            }
            carry += total;
        }
    }
    __syncthreads();

    Place at = {}, ahead;
    int units = x1 - x0, first = 0;                       // first: where the current (sequence, head) begins in the list
    if (units > 0) {
        at.b = s_b[w];
        at.len = seq_len(p.q, at.b, p.status);
        at.nch = (at.len + 15) >> 4;
        const int rel = x0 - s_pre[w];
        at.vh = rel / at.nch;
        at.c = rel - at.vh * at.nch;
        first = x0 - at.c;
    }
    ahead = at;

    // ---- loading
    uint8_t* ring = smem + (size_t)w * NST * S::UNIT;
    const uint32_t ring_u = tq_smem_u32(ring);
    const bool whole = (p.g.page & 15) == 0;              // a unit lies in one page
    const int page_units = whole ? p.g.page >> 4 : 1;
    int tab_b = -1, tab_c = 0, tab = 0, tab_next = 0;     // lane i: table entries of chunks tab_c + i and tab_c + 32 + i
    auto entry = [&](int chunk) {
        return chunk < ahead.nch ? p.q.table[(int64_t)ahead.b * p.q.table_stride + chunk / page_units] : 0;
    };
    auto issue = [&](int stage) {
        const int t0 = ahead.c << 4, left = ahead.len - t0;
        const int head = ahead.vh / p.RT;
        const uint32_t dst = ring_u + stage * S::UNIT;
        uint32_t mask = left >= 16 ? 0xffffu : (1u << left) - 1u;
        const int r0 = lane / LPR, ch = lane % LPR;
        if (whole) {
            if (ahead.b != tab_b || ahead.c < tab_c || ahead.c >= tab_c + 64) {
                tab_b = ahead.b;
                tab_c = ahead.c;
                tab = entry(tab_c + lane);
                tab_next = entry(tab_c + 32 + lane);
            } else if (ahead.c >= tab_c + 32) {
                tab_c += 32;
                tab = tab_next;
                tab_next = entry(tab_c + 32 + lane);
            }
            const int e = __shfl_sync(0xffffffffu, tab, ahead.c - tab_c);
            const bool ok = (uint32_t)e < (uint64_t)p.g.num_blocks;
            if (!ok) {
                mask = 0;
                if (lane == 0) atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
            }
            const int64_t off = (ok ? (int64_t)e : 0) * p.g.sb + (int64_t)((ahead.c % page_units) << 4) * p.g.st + head * p.g.sh + ch * 16;
            const uint8_t *k = p.g.k + off, *v = p.g.v + off;
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) {
                const int r = i * RPI + r0;
                const bool there = (mask >> r) & 1;
                const uint32_t d = dst + r * ROWB + ((ch ^ (r & 7)) << 4);
                const int64_t o = there ? r * p.g.st : 0;
                cp_async16(d, k + o, there);
                cp_async16(d + 16 * ROWB, v + o, there);
            }
        } else {                                          // pages end anywhere: a table entry per row
            const int r = lane & 15, t = t0 + r;
            int64_t off = 0;
            bool ok = false;
            if (r < left) {
                const int e = p.q.table[(int64_t)ahead.b * p.q.table_stride + t / p.g.page];
                ok = (uint32_t)e < (uint64_t)p.g.num_blocks;
                if (ok) off = (int64_t)e * p.g.sb + (int64_t)(t % p.g.page) * p.g.st + head * p.g.sh;
                else atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
            }
            mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) {
                const int rr = i * RPI + r0;
                const int64_t o = __shfl_sync(0xffffffffu, off, rr) + ch * 16;
                const bool there = (mask >> rr) & 1;
                const uint32_t d = dst + rr * ROWB + ((ch ^ (rr & 7)) << 4);
                cp_async16(d, p.g.k + o, there);
                cp_async16(d + 16 * ROWB, p.g.v + o, there);
            }
        }
        if (lane == 0) s_mask[w][stage] = mask;
    };

    int issued = 0;
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) {
        if (issued < units) {
            issue(i);
            if (++issued < units) advance(ahead, p, VH);
        }
        cp_async_commit();
    }

    // ---- the current (sequence, head)
    uint32_t qf[NT][KS][2];
    float acc[KS][NT][4], m[NT][2], l[NT][2];
    auto rows_of = [&](int vh) { return min(p.G - (vh % p.RT) * 8 * NT, 8 * NT); };       // query heads of this row tile
    auto first_row = [&](int b, int vh) { return (int64_t)b * p.Qh + (vh / p.RT) * p.G + (vh % p.RT) * 8 * NT; };
    auto begin = [&]() {
        const int rows = rows_of(at.vh);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint8_t* q = p.query + (first_row(at.b, at.vh) + nt * 8 + g) * ROWB + t4 * 4;
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
    auto write_out = [&](int b, int vh) {                 // l summed
        const int rows = rows_of(vh);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float i0 = l[nt][0] == 0.f ? 0.f : 1.f / l[nt][0], i1 = l[nt][1] == 0.f ? 0.f : 1.f / l[nt][1];
            uint8_t* o = p.out + (first_row(b, vh) + nt * 8 + g) * ROWB + t4 * 4;
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
                        p.lse[first_row(b, vh) + nt * 8 + 2 * t4 + j] = l[nt][j] == 0.f ? INFINITY : m[nt][j] + log2f(l[nt][j]);
        }
    };
    auto write_slot = [&](float* slot) {                  // l summed
        float4* s = reinterpret_cast<float4*>(slot);
#pragma unroll
        for (int ct = 0; ct < KS; ++ct)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s[(ct * NT + nt) * 32 + lane] = make_float4(acc[ct][nt][0], acc[ct][nt][1], acc[ct][nt][2], acc[ct][nt][3]);
        if (g == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[S::ACC4 + nt * 4 + t4] = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
    };
    auto add_slot = [&](const float* slot) {
        const float4* s = reinterpret_cast<const float4*>(slot);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
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
    auto note_event = [&](int which) {
        if (lane == 0) s_event[which] = Event{1, at.b, at.vh, first, at.nch};
    };

    // flags: 0 no units; 1 this warp's first piece ends a (sequence, head) that an earlier warp began; 2 its whole share is such a
    // piece and goes on; 3 begins with a (sequence, head) of its own
    int flag = 0;
    bool open = false;          // the last piece goes on behind this warp's share
    if (units > 0) {
        flag = at.c == 0 ? 3 : (at.nch - at.c <= units ? 1 : 2);
        begin();
    }
    const uint32_t k_row = (((lane >> 3) & 1) * 8 + (lane & 7)), k_ch = lane >> 4;      // ldmatrix: row and chunk of this lane's address
    const uint32_t v_row = ((lane >> 4) * 8 + (lane & 7)), v_ch = (lane >> 3) & 1;
#pragma unroll 1
    for (int u = 0; u < units; ++u) {
        cp_async_wait<NST - 2>();
        __syncwarp();
        if (issued < units) {
            issue((u + NST - 1) % NST);
            if (++issued < units) advance(ahead, p, VH);
        }
        cp_async_commit();

        const uint32_t kb = ring_u + (u % NST) * S::UNIT, vb = kb + 16 * ROWB;
        const uint32_t mask = s_mask[w][u % NST];
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t a[4];
            ldsm4(a, kb + k_row * ROWB + (((ks * 2 + k_ch) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<BF16>(ks & 1 ? s2[nt] : s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[nt][i] = (s[nt][i] + s2[nt][i]) * p.scale_log2;
                if (!((mask >> (g + (i >> 1) * 8)) & 1)) s[nt][i] = -INFINITY;
            }
            grows |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] || fmaxf(s[nt][1], s[nt][3]) > m[nt][1];
        }
        if (p.scores != nullptr) {
            const int rows = rows_of(at.vh);
            float* sc = p.scores + first_row(at.b, at.vh) * p.score_stride + at.c * 16 + g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = nt * 8 + 2 * t4 + (i & 1);
                    if (row < rows) sc[row * p.score_stride + (i >> 1) * 8] = s[nt][i];
                }
        }
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
                const float a = ex2(s[nt][2 * k] - r0), c = ex2(s[nt][2 * k + 1] - r1);
                l[nt][0] += a;
                l[nt][1] += c;
                const uint32_t h = pack<BF16>(a, c);
                const float2 back = unpack<BF16>(h);
                hi[nt][k] = transpose8(h);
                rest[nt][k] = transpose8(pack<BF16>(a - back.x, c - back.y));
            }
        }
#pragma unroll
        for (int ct = 0; ct < KS; ++ct) {
            uint32_t a[4];
            ldsm4t(a, vb + v_row * ROWB + (((ct * 2 + v_ch) ^ (v_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma<BF16>(acc[ct][nt], a, hi[nt][0], hi[nt][1]);
                mma<BF16>(acc[ct][nt], a, rest[nt][0], rest[nt][1]);
            }
        }

        const bool ends = at.c + 1 == at.nch;
        if (ends) {
            sum_l();
            const bool began_here = first >= x0;
            if (began_here) {
                write_out(at.b, at.vh);
            } else if (w > 0) {
                write_slot(slots + w * S::SLOT);
            } else {                                      // the piece of an earlier CTA ends in this one's first warp
                write_slot(global_slot(blockIdx.x, 0));
                note_event(0);
            }
        }
        if (u + 1 < units) {
            advance(at, p, VH);
            if (ends) {
                first = x0 + u + 1;
                begin();
            }
        } else {
            open = !ends;
        }
    }
    cp_async_wait<0>();
    if (open) {
        sum_l();
        if (flag == 2 && w > 0) write_slot(slots + w * S::SLOT);
    }
    if (lane == 0) s_flag[w] = flag;
    __syncthreads();

    // ---- join the pieces of this CTA's warps: the warp that holds the first piece adds the others in order
    if (open && !(flag == 2 && w > 0)) {
        bool done = false;
        for (int i = w + 1; i < NW && !done; ++i) {
            const int f = s_flag[i];
            if (f == 0) continue;
            if (f == 3) break;                            // cannot be: an open piece goes on in the next warp that has units
            add_slot(slots + i * S::SLOT);
            done = f == 1;
        }
        if (done && first >= lo) {
            write_out(at.b, at.vh);
        } else {
            const int which = first >= lo ? 1 : 0;
            write_slot(global_slot(blockIdx.x, which));
            note_event(which);
        }
    }
    __syncthreads();

    // ---- join across CTAs: the last to arrive adds up all pieces in the order of the list
    if (!s_event[0].valid && !s_event[1].valid) return;
    if (tid == 0) {
        __threadfence();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            s_last[e] = 0;
            if (!s_event[e].valid) continue;
            const int from = s_event[e].first / share, to = (s_event[e].first + s_event[e].nch - 1) / share;
            if (atomicAdd(&p.tickets[from], 1) == to - from) {
                p.tickets[from] = 0;                      // for the next launch
                s_last[e] = 1;
            }
        }
        __threadfence();
    }
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
        if (!s_last[e]) continue;
        const Event ev = s_event[e];
        const int from = ev.first / share, pieces = (ev.first + ev.nch - 1) / share - from + 1;
        auto piece = [&](int i) { return reinterpret_cast<const float4*>(global_slot(from + i, i == 0 ? 1 : 0)); };
        float* wt = reinterpret_cast<float*>(smem);       // [pieces][8 NT] weights of the pieces
        const int rows = rows_of(ev.vh);
        const int64_t row0 = first_row(ev.b, ev.vh);
        for (int r = w; r < 8 * NT; r += NW) {
            const int j = r & 1;
            float mx = -INFINITY, sum = 0.f;
            for (int i = lane; i < pieces; i += 32) {
                const float4 ml = __ldcg(piece(i) + S::ACC4 + (r >> 1));
                mx = fmaxf(mx, j ? ml.y : ml.x);
            }
            mx = tq_warp_max(mx);
            for (int i = lane; i < pieces; i += 32) {
                const float4 ml = __ldcg(piece(i) + S::ACC4 + (r >> 1));
                const float a = weight(j ? ml.y : ml.x, mx);
                wt[i * 8 * NT + r] = a;
                sum += a * (j ? ml.w : ml.z);
            }
            sum = tq_warp_sum(sum);
            if (lane == 0) {
                s_inv[r] = sum == 0.f ? 0.f : 1.f / sum;
                if (p.lse != nullptr && r < rows) p.lse[row0 + r] = sum == 0.f ? INFINITY : mx + log2f(sum);
            }
        }
        __syncthreads();
        for (int f = tid; f < S::ACC4; f += S::THREADS) {
            const int ln = f & 31, nt = (f >> 5) % NT, ct = (f >> 5) / NT;
            const int row = nt * 8 + 2 * (ln & 3), chan = ct * 16 + (ln >> 2);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int i = 0; i < pieces; ++i) {
                const float4 v = __ldcg(piece(i) + f);
                const float2 k = *reinterpret_cast<const float2*>(wt + i * 8 * NT + row);
                a.x = fmaf(v.x, k.x, a.x);
                a.y = fmaf(v.y, k.y, a.y);
                a.z = fmaf(v.z, k.x, a.z);
                a.w = fmaf(v.w, k.y, a.w);
            }
            const float i0 = s_inv[row], i1 = s_inv[row + 1];
            using E = TqElem<BF16 ? TQ_BF16 : TQ_F16>;
            if (row < rows) {
                E::store(p.out, (row0 + row) * D + chan, a.x * i0);
                E::store(p.out, (row0 + row) * D + chan + 8, a.z * i0);
            }
            if (row + 1 < rows) {
                E::store(p.out, (row0 + row + 1) * D + chan, a.y * i1);
                E::store(p.out, (row0 + row + 1) * D + chan + 8, a.w * i1);
            }
        }
        __syncthreads();
    }
}

// mass[b][h][t] += sum over the group's heads of 2^(score - lse): 4 G bytes read and 8 moved a token and head, against the 4 D
// that the attention reads.
__global__ void __launch_bounds__(256) tq_pages_ledger_kernel(const Batch q, const float* __restrict__ scores, int64_t score_stride,
                                                              const float* __restrict__ lse, int H, int G, float* mass,
                                                              int64_t mass_stride, int32_t* status) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = blockIdx.x / H, t = blockIdx.y * 256 + threadIdx.x;
    if (t >= seq_len(q, b, status)) return;
    const int64_t row = (int64_t)blockIdx.x * G;
    float sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < G; ++i) sum += ex2(__ldcs(scores + (row + i) * score_stride + t) - lse[row + i]);
    mass[blockIdx.x * mass_stride + t] += sum;
}

struct Scratch {
    size_t partials, lse, scores, bytes;
    int64_t score_stride;
};
int row_tiles(int G) { return (G + 15) / 16; }
Scratch scratch_of(const tq_pages* g, const tq_pages_batch* q, int Qh, bool ledger) {
    const int nt = Qh / g->num_kv_heads > 8 ? 2 : 1;
    const size_t slot = (size_t)g->head_dim / 16 * nt * 128 + nt * 16;
    Scratch s;
    s.partials = 0;
    s.lse = (size_t)tq_sm_count() * 2 * slot * 4;
    s.score_stride = ((int64_t)q->max_seq_len + 15) / 16 * 16;
    s.scores = s.lse + (ledger ? ((size_t)q->batch * Qh * 4 + 255) / 256 * 256 : 0);
    s.bytes = s.scores + (ledger ? (size_t)q->batch * Qh * s.score_stride * 4 : 0);
    return s;
}

template <int D, int NT, bool BF16>
int launch(const DecodeParams& p, int ctas, cudaStream_t st) {
    using S = Shape<D, NT>;
    static TqSmemOptIn opt_in;
    if (tq_opt_in_smem(tq_pages_decode_kernel<D, NT, BF16>, S::SMEM, opt_in) != TQ_OK) return TQ_ERR_CUDA;
    tq_pages_decode_kernel<D, NT, BF16><<<ctas, S::THREADS, S::SMEM, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? TQ_OK : TQ_ERR_CUDA;
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
    if (heads * q->batch * (((int64_t)q->max_seq_len + 15) / 16) >= ((int64_t)1 << 31)) return TQ_ERR_SHAPE;
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
    if (mass && batch->max_seq_len > 65535 * 256) return TQ_ERR_SHAPE;      // a grid's second dimension
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
    const int ctas = tq_sm_count(), two = p.G > 8;
    tq_note_launch(st, TQ_LAUNCH_WAITED);
    switch (pages->head_dim) {
        case 64: rc = two ? launch_dtype<64, 2>(p, pages->dtype, ctas, st) : launch_dtype<64, 1>(p, pages->dtype, ctas, st); break;
        case 128: rc = two ? launch_dtype<128, 2>(p, pages->dtype, ctas, st) : launch_dtype<128, 1>(p, pages->dtype, ctas, st); break;
        default: rc = two ? launch_dtype<256, 2>(p, pages->dtype, ctas, st) : launch_dtype<256, 1>(p, pages->dtype, ctas, st); break;
    }
    if (rc != TQ_OK || !mass) return rc;
    const dim3 grid((unsigned)(batch->batch * pages->num_kv_heads), (unsigned)((batch->max_seq_len + 255) / 256));
    tq_pages_ledger_kernel<<<grid, 256, 0, st>>>(p.q, p.scores, p.score_stride, p.lse, pages->num_kv_heads, p.G, mass, mass_stride, status);
    return cudaGetLastError() == cudaSuccess ? TQ_OK : TQ_ERR_CUDA;
}
