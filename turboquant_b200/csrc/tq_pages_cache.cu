// The exact paged cache without its attention: writing tokens into the pages, and evicting the tokens that received least.
#include "tq_pages.cuh"

using namespace tqpg;

namespace {

// ---------------------------------------------------------------------------------------------------------------- write

// A copy, bound by HBM (4 D bytes a token and head read, as many written).  A CTA takes WR_TOK tokens at a time, thread by
// thread 16 bytes of key and value of each, all loads before the first store.
constexpr int WR_THREADS = 256, WR_TOK = 4;

struct WriteParams {
    Pages g;
    const uint8_t *k, *v;
    int64_t kt, kh, vt, vh;    // bytes
    int64_t n;
    const int64_t* slots;
    int32_t* status;
};

template <int D>
__global__ void __launch_bounds__(WR_THREADS) tq_pages_write_kernel(const WriteParams p) {
    constexpr int CH = D / 8;                              // 16-byte pieces of a row
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int pieces = p.g.H * CH;
    const int64_t t0 = (int64_t)blockIdx.x * WR_TOK;
    for (int i = threadIdx.x; i < 2 * pieces; i += WR_THREADS) {
        const bool value = i >= pieces;
        const int j = value ? i - pieces : i, h = j / CH, c = (j % CH) * 16;
        const uint8_t* src = (value ? p.v + h * p.vh : p.k + h * p.kh) + c;
        uint8_t* dst = (value ? p.g.v : p.g.k) + h * p.g.sh + c;
        const int64_t step = value ? p.vt : p.kt;
        uint4 x[WR_TOK];
        int64_t slot[WR_TOK];
#pragma unroll
        for (int t = 0; t < WR_TOK; ++t) {
            slot[t] = t0 + t < p.n ? p.slots[t0 + t] : -1;
            if (t0 + t < p.n) x[t] = __ldcs(reinterpret_cast<const uint4*>(src + (t0 + t) * step));
        }
#pragma unroll
        for (int t = 0; t < WR_TOK; ++t) {
            if (slot[t] < 0) continue;
            const int64_t block = slot[t] / p.g.page;
            if (block >= p.g.num_blocks) {
                atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
                continue;
            }
            *reinterpret_cast<uint4*>(dst + block * p.g.sb + (slot[t] - block * p.g.page) * p.g.st) = x[t];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- evict

// One CTA settles a (sequence, kv head): which slots are kept, the ledger, and the list of moves; a second launch moves the
// rows.  Order of keeping: protected tokens, then mass as a 32-bit key with the order of the numbers.  The k-th largest key is
// found bit by bit, from the highest one in which the candidates differ, by counting the keys that reach a trial value - no
// histogram, so nothing depends on how the weights spread (they differ by a few powers of two, and the counters of a histogram
// would be hit by all lanes at once).  A trial costs two instructions a key and one exchange between the warps.  Lane-striped
// slots (warp * 32 * KPT + i * 32 + lane) let a ballot count a row and keep every list in ascending order.
struct EvictParams {
    Pages g;
    Batch q;
    const float* mass;
    const int32_t* positions;
    const int32_t *held, *seen;
    float* out_mass;
    int32_t* out_positions;
    int32_t *out_held, *out_seen, *new_lens;
    int64_t stride, out_stride;    // max_tokens
    int budget, recent;
    int32_t* dst;                  // [batch * H][list]
    int32_t* src;
    int32_t* count;                // [batch * H]
    int list;
    int32_t* status;
};

// order of the floats: NaN above everything, -0 like 0; never 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exchange of one number a warp; two buffers in turn, one barrier.
struct CtaSum {
    int* buf;      // [2][32]
    int turn, warps;
    __device__ __forceinline__ int all_of(int x) {         // what the lane's warp gave
        int* b = buf + (turn & 1) * 32;
        turn ^= 1;
        const int lane = threadIdx.x & 31;
        if (lane == 0) b[threadIdx.x >> 5] = x;
        __syncthreads();
        return lane < warps ? b[lane] : 0;
    }
    __device__ __forceinline__ int operator()(int x) { return __reduce_add_sync(0xffffffffu, all_of(x)); }
    // the sum of the warps before this one, and of all
    __device__ __forceinline__ int before(int x, int& total) {
        const int y = all_of(x), lane = threadIdx.x & 31;
        total = __reduce_add_sync(0xffffffffu, y);
        return __reduce_add_sync(0xffffffffu, lane < (int)(threadIdx.x >> 5) ? y : 0);
    }
};

// KPT slots a thread, held as keys in registers; a row that is longer than all threads hold (LONG) is gone over again for every
// count.  Masses and positions are read again where they are written: they are in the caches.
template <int KPT, bool LONG>
__global__ void __launch_bounds__(1024) tq_pages_evict_kernel(const EvictParams p) {
    __shared__ int s_buf[64];
    const int row = blockIdx.x, b = row / p.g.H, lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t below = (1u << lane) - 1u;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int n = seq_len(p.q, b, p.status), m = min(n, p.budget);
    const int held = p.held[b], seen = p.seen[b], late = seen + n - held - p.recent;
    const float* mass = p.mass + row * p.stride;
    const int32_t* positions = p.positions + row * p.stride;
    float* out_mass = p.out_mass + row * p.out_stride;
    int32_t* out_positions = p.out_positions + row * p.out_stride;
    int32_t *dst = p.dst + (int64_t)row * p.list, *src = p.src + (int64_t)row * p.list;
    CtaSum sum{s_buf, 0, warps};
    const int span = warps * 32 * KPT, rounds = LONG ? (n + span - 1) / span : 1;

    uint32_t key[KPT];                 // 0: not in the cache
    uint32_t guard = 0;                // bit i: slot i of this thread is protected
    auto slot_of = [&](int r, int i) { return r * span + (w * KPT + i) * 32 + lane; };
    auto position = [&](int t) { return t < held ? positions[t] : seen + t - held; };
    auto load = [&](int r) {
        const int t0 = slot_of(r, 0);
        guard = 0;
#pragma unroll
        for (int c = 0; c < KPT; c += 8) {                 // eight at a time: more would not fit the registers
            float x[8];
            int pos[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = t0 + (c + i) * 32 < n ? mass[t0 + (c + i) * 32] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) pos[i] = t0 + (c + i) * 32 < n ? position(t0 + (c + i) * 32) : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool there = t0 + (c + i) * 32 < n;
                key[c + i] = there ? key_of(x[i]) : 0u;
                guard |= (uint32_t)(there && pos[i] >= late) << (c + i);
            }
            asm volatile("" ::: "memory");
        }
    };
    load(0);

    // protected tokens first; the rest by key, or the protected by key where they alone exceed the budget
    const bool trims = n > m;
    bool all_guarded = false;          // the candidates are the protected tokens
    uint32_t limit = 0u;               // the k-th largest key of the candidates
    int equal_taken = 0;               // how many of the keys equal to it are taken, lowest slots first
    auto among = [&](int i) { return ((guard >> i) & 1u) == (uint32_t)all_guarded; };
    if (trims) {
        int guarded = 0;
        for (int r = 0; r < rounds; ++r) {
            if (LONG && r > 0) load(r);
            guarded += __popc(guard);
        }
        guarded = sum(__reduce_add_sync(0xffffffffu, guarded));
        all_guarded = guarded >= m;
        const int k = all_guarded ? m : m - guarded;
        // keys of others than candidates are 0 from here on, and no trial value is
        uint32_t ones = 0xffffffffu, any = 0u;
        auto drop = [&]() {
#pragma unroll
            for (int i = 0; i < KPT; ++i)
                if (!among(i)) key[i] = 0u;
        };
        for (int r = 0; r < rounds; ++r) {
            if (LONG) load(r);
            drop();
#pragma unroll
            for (int i = 0; i < KPT; ++i)
                if (key[i] != 0u) ones &= key[i], any |= key[i];
        }
        ones = (uint32_t)sum.all_of((int)__reduce_and_sync(0xffffffffu, ones));
        any = (uint32_t)sum.all_of((int)__reduce_or_sync(0xffffffffu, any));
        ones = __reduce_and_sync(0xffffffffu, lane < warps ? ones : 0xffffffffu);
        any = __reduce_or_sync(0xffffffffu, any);
        const uint32_t differ = ones ^ any;
        int bit = 31 - __clz(differ), reach = -1;          // reach: keys >= limit
        limit = differ == 0u ? any : bit == 31 ? 0u : any >> (bit + 1) << (bit + 1);       // what all candidates have in common
        for (; bit >= 0 && reach != k; --bit) {
            const uint32_t trial = limit | (1u << bit);
            int c = 0;
            for (int r = 0; r < rounds; ++r) {
                if (LONG) {
                    load(r);
                    drop();
                }
#pragma unroll
                for (int i = 0; i < KPT; ++i) c += key[i] >= trial;
            }
            c = sum(__reduce_add_sync(0xffffffffu, c));
            if (c >= k) {
                limit = trial;
                reach = c;
            }
        }
        if (k == 0) {                                      // nothing but the protected ones
            limit = 0xffffffffu;
        } else if (reach == k) {
            equal_taken = 0x7fffffff;
        } else {
            int above = 0;
            for (int r = 0; r < rounds; ++r) {
                if (LONG) {
                    load(r);
                    drop();
                }
#pragma unroll
                for (int i = 0; i < KPT; ++i) above += key[i] > limit;
            }
            equal_taken = k - sum(__reduce_add_sync(0xffffffffu, above));
        }
    }

    // the lists, in ascending order: holes before m, movers behind it
    int equals = 0, holes = 0, movers = 0;                 // of the slots before this round
    for (int r = 0; r < rounds; ++r) {
        if (LONG) {
            load(r);
            if (trims) {
#pragma unroll
                for (int i = 0; i < KPT; ++i)
                    if (!among(i)) key[i] = 0u;
            }
        }
        const int t0 = slot_of(r, 0);
        int mine = 0, total;
        if (trims) {
#pragma unroll
            for (int i = 0; i < KPT; ++i) mine += __popc(__ballot_sync(0xffffffffu, key[i] != 0u && key[i] == limit));
        }
        int rank = equals + sum.before(mine, total);
        equals += total;
        uint32_t kept = 0;                                 // bit i: slot i of this thread stays in the cache
        int my_holes = 0, my_movers = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            bool stays = t < n;
            if (trims) {
                const uint32_t eq = __ballot_sync(0xffffffffu, key[i] != 0u && key[i] == limit);
                stays = stays && (among(i) ? key[i] > limit || (key[i] == limit && rank + __popc(eq & below) < equal_taken) : !all_guarded);
                rank += __popc(eq);
            }
            my_holes += __popc(__ballot_sync(0xffffffffu, t < m && !stays));
            my_movers += __popc(__ballot_sync(0xffffffffu, t >= m && stays));
            kept |= (uint32_t)stays << i;
        }
        int total_holes, total_movers;
        int hole_at = holes + sum.before(my_holes, total_holes), mover_at = movers + sum.before(my_movers, total_movers);
        holes += total_holes;
        movers += total_movers;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            const bool stays = (kept >> i) & 1;
            const uint32_t hole = __ballot_sync(0xffffffffu, t < m && !stays);
            if (t < m && !stays) dst[hole_at + __popc(hole & below)] = t;
            hole_at += __popc(hole);
            if (t < m && stays) {
                out_mass[t] = mass[t];
                out_positions[t] = position(t);
            }
        }
        __syncthreads();                                   // every hole that a mover of this round takes has been noted: holes lie before movers
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            const bool moves = t >= m && ((kept >> i) & 1);
            const uint32_t mover = __ballot_sync(0xffffffffu, moves);
            if (moves) {
                const int j = mover_at + __popc(mover & below), to = dst[j];
                src[j] = t;
                out_mass[to] = mass[t];
                out_positions[to] = position(t);
            }
            mover_at += __popc(mover);
        }
    }
    __syncthreads();                                       // in place: nothing is cleared before it has been read
    for (int64_t t = m + (int)threadIdx.x; t < p.out_stride; t += blockDim.x) {
        out_mass[t] = 0.f;
        out_positions[t] = -1;
    }
    if (threadIdx.x == 0) p.count[row] = holes;
}

// The moves of all (sequence, kv head) rows: a group of D/8 lanes copies a key row, then a value row.
template <int D>
__global__ void __launch_bounds__(256) tq_pages_move_kernel(const EvictParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int LPR = D / 8, PER = 256 / LPR;
    const int row = blockIdx.x, b = row / p.g.H, h = row % p.g.H;
    if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0) {   // here, not in the first launch: other heads of the sequence read them there
        const int n = seq_len(p.q, b, p.status), held = p.held[b], seen = p.seen[b];
        p.new_lens[b] = min(n, p.budget);
        p.out_seen[b] = seen + n - held;
        p.out_held[b] = min(n, p.budget);
    }
    const int count = p.count[row];
    const int32_t* table = p.q.table + (int64_t)b * p.q.table_stride;
    for (int j = blockIdx.y * PER + threadIdx.x / LPR; j < count; j += gridDim.y * PER) {
        const int from = p.src[(int64_t)row * p.list + j], to = p.dst[(int64_t)row * p.list + j];
        const int eb = table[from / p.g.page], tb = table[to / p.g.page];
        if ((uint32_t)eb >= (uint64_t)p.g.num_blocks || (uint32_t)tb >= (uint64_t)p.g.num_blocks) {
            atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
            continue;
        }
        const int64_t o = (threadIdx.x % LPR) * 16 + h * p.g.sh;
        const int64_t s = eb * p.g.sb + (from % p.g.page) * p.g.st + o, d = tb * p.g.sb + (to % p.g.page) * p.g.st + o;
        const uint4 k = *reinterpret_cast<const uint4*>(p.g.k + s), v = *reinterpret_cast<const uint4*>(p.g.v + s);
        *reinterpret_cast<uint4*>(p.g.k + d) = k;
        *reinterpret_cast<uint4*>(p.g.v + d) = v;
    }
}

int evict_list(const tq_pages_batch* q, int budget) {      // moves of a row at most
    const int behind = q->max_seq_len - budget;
    return behind <= 0 ? 0 : behind < budget ? behind : budget;
}
int evict_check(const tq_pages* g, const tq_pages_batch* q, int budget) {
    int rc = pages_check(g);
    if (rc == TQ_OK) rc = batch_check(g, q);
    if (rc == TQ_OK && (budget < 0 || (int64_t)q->batch * g->num_kv_heads >= ((int64_t)1 << 31))) rc = TQ_ERR_SHAPE;
    return rc;
}

}  // namespace

extern "C" int tq_pages_write(const tq_pages* pages, const void* key, const void* value, int64_t n_tokens, int64_t key_stride_token,
                              int64_t key_stride_head, int64_t value_stride_token, int64_t value_stride_head, const int64_t* slot_mapping,
                              int32_t* status, void* stream) {
    const int rc = pages_check(pages);
    if (rc != TQ_OK) return rc;
    if (n_tokens < 0) return TQ_ERR_SHAPE;
    if (n_tokens == 0) return TQ_OK;
    if (!key || !value || !slot_mapping || !status) return TQ_ERR_NULL;
    if (((uintptr_t)key & 15) || ((uintptr_t)value & 15) || (key_stride_token & 7) || (key_stride_head & 7) || (value_stride_token & 7) ||
        (value_stride_head & 7))
        return TQ_ERR_ALIGN;
    const int64_t ctas = (n_tokens + WR_TOK - 1) / WR_TOK;
    if (ctas >= ((int64_t)1 << 31)) return TQ_ERR_SHAPE;
    const WriteParams p{pages_of(pages), static_cast<const uint8_t*>(key), static_cast<const uint8_t*>(value), key_stride_token * 2,
                        key_stride_head * 2, value_stride_token * 2, value_stride_head * 2, n_tokens, slot_mapping, status};
    cudaStream_t st = (cudaStream_t)stream;
    tq_note_launch(st, TQ_LAUNCH_WAITED);      // writes rows that a store may read next
    switch (pages->head_dim) {
        case 64: return launch_behind(tq_pages_write_kernel<64>, dim3((unsigned)ctas), WR_THREADS, 0, st, p);
        case 128: return launch_behind(tq_pages_write_kernel<128>, dim3((unsigned)ctas), WR_THREADS, 0, st, p);
        default: return launch_behind(tq_pages_write_kernel<256>, dim3((unsigned)ctas), WR_THREADS, 0, st, p);
    }
}

extern "C" int tq_pages_evict_scratch_bytes(const tq_pages* pages, const tq_pages_batch* batch, int32_t budget, size_t* out) {
    if (!out) return TQ_ERR_NULL;
    const int rc = evict_check(pages, batch, budget);
    if (rc != TQ_OK) return rc;
    const size_t rows = (size_t)batch->batch * pages->num_kv_heads;
    *out = rows * 4 + rows * evict_list(batch, budget) * 8;
    return TQ_OK;
}

extern "C" int tq_pages_evict(const tq_pages* pages, const tq_pages_batch* batch, const tq_pages_ledger* ledger, const tq_pages_ledger* out,
                              int32_t budget, int32_t recent, int32_t* new_lens, void* scratch, size_t scratch_bytes, int32_t* status,
                              void* stream) {
    size_t need = 0;
    const int rc = tq_pages_evict_scratch_bytes(pages, batch, budget, &need);
    if (rc != TQ_OK) return rc;
    if (!ledger || !out || !new_lens || !scratch || !status) return TQ_ERR_NULL;
    for (const tq_pages_ledger* l : {ledger, out}) {
        if (!l->mass || !l->positions || !l->held || !l->seen) return TQ_ERR_NULL;
        if (l->max_tokens < batch->max_seq_len) return TQ_ERR_RANGE;
    }
    if (recent < 0 || recent > budget) return TQ_ERR_SHAPE;
    if (scratch_bytes < need) return TQ_ERR_WORKSPACE;
    if ((uintptr_t)scratch & 15) return TQ_ERR_ALIGN;
    const int64_t rows = (int64_t)batch->batch * pages->num_kv_heads;
    EvictParams p;
    p.g = pages_of(pages);
    p.q = batch_of(batch);
    p.mass = ledger->mass;
    p.positions = ledger->positions;
    p.held = ledger->held;
    p.seen = ledger->seen;
    p.out_mass = out->mass;
    p.out_positions = out->positions;
    p.out_held = out->held;
    p.out_seen = out->seen;
    p.new_lens = new_lens;
    p.stride = ledger->max_tokens;
    p.out_stride = out->max_tokens;
    p.budget = budget;
    p.recent = recent;
    p.list = evict_list(batch, budget);
    p.count = static_cast<int32_t*>(scratch);
    p.dst = p.count + rows;
    p.src = p.dst + rows * p.list;
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    tq_note_launch(st, TQ_LAUNCH_WAITED);      // writes rows that a store may read next
    const int n = batch->max_seq_len;
    auto threads_for = [&](int kpt) { return n >= 1024 * kpt ? 1024 : (n + 32 * kpt - 1) / (32 * kpt) * 32; };
    int rc2;
    // eight keys a thread as far as 1024 threads hold the row, then thirty-two
    if (n <= 1024 * 8) rc2 = launch_behind(tq_pages_evict_kernel<8, false>, dim3((unsigned)rows), threads_for(8), 0, st, p);
    else if (n <= 1024 * 32) rc2 = launch_behind(tq_pages_evict_kernel<32, false>, dim3((unsigned)rows), threads_for(32), 0, st, p);
    else rc2 = launch_behind(tq_pages_evict_kernel<32, true>, dim3((unsigned)rows), 1024, 0, st, p);
    if (rc2 != TQ_OK) return rc2;
    const int per = 256 / (pages->head_dim / 8);
    const int64_t tiles = (p.list + per - 1) / per;
    const dim3 grid((unsigned)rows, (unsigned)(tiles < 1 ? 1 : tiles > 1024 ? 1024 : tiles));
    switch (pages->head_dim) {
        case 64: return launch_behind(tq_pages_move_kernel<64>, grid, 256, 0, st, p);
        case 128: return launch_behind(tq_pages_move_kernel<128>, grid, 256, 0, st, p);
        default: return launch_behind(tq_pages_move_kernel<256>, grid, 256, 0, st, p);
    }
}
