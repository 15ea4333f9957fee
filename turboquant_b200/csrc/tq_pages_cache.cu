// The exact paged cache without its attention: writing tokens into the pages, and evicting the tokens that received least.
#include "tq_pages.cuh"

using namespace tqpg;

namespace {

// ---------------------------------------------------------------------------------------------------------------- write

// A copy, bound by HBM (4 D bytes a token and head read, as many written).  A CTA takes WR_TOK tokens at a time, thread by
// thread 16 bytes of key and value of each, all loads before the first store.  32768 tokens of 8 heads of 128, 268 MB: 42.5 us,
// 6.3 TB/s; 64 tokens 2.9 us, the launch.
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

// A team of CTAs - one, or a cluster of up to eight - settles a (sequence, kv head): which slots are kept, the ledger, and the list
// of moves; a second launch moves the rows.  Order of keeping: protected tokens, then mass as a 32-bit key with the order of the
// numbers.  The k-th largest key lies between two keys of the row; a trial in the middle counts those that reach it and finds
// the nearest keys on either side of it, which become the new ends.  Nothing depends on how the weights spread (a histogram's
// counters would be hit by all lanes at once: they differ by a few powers of two), and equal keys end the search.  Once few keys
// are left between the ends, one warp settles those alone.  Lane-striped slots (warp * 32 * KPT + i * 32 + lane) let a ballot
// count a row and keep every list in ascending order.
//
// A token that moves goes into a list with its mass and position; the second launch, which needs the list for the rows, puts them in
// their places (in this one a mover would have to wait for the holes of the other CTAs: 1.1 us more for 512 rows of 2112, 1.6 for
// 32 of up to 32768, 2.7 for one of 32768).
//
// Bound by the chain of loads, exchanges and lists.  Both launches take 9.6 us for 300 slots, 19.3 for 512 rows of 2112, of which
// moving the rows is 8 (four CTAs an SM at 56 registers; at 40 they spill and it is 16 longer), 43.5 for 32 rows of up to 32768 in
// clusters of four, of which moving is 20 (a cluster's exchange takes 1.6 us, a CTA's 0.2: candidates go to one CTA as soon as it
// holds them).
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
    float* src_mass;               // of the tokens that move
    int32_t* src_positions;
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

constexpr int EV_KPT = 8, EV_WARPS = 32, EV_CTAS = 8;      // slots a thread, warps a CTA and CTAs a team at most
constexpr int EV_SOME = EV_WARPS * 32 * EV_KPT, EV_FEW = 128;      // keys that a team's first CTA, and that one warp settles alone

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void put_in_cta(uint32_t addr, const uint4& x) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}

// Exchange of numbers between the warps of a CTA and, in a TEAM, between the CTAs of a cluster: two buffers in turn each, a
// barrier of each kind (the cluster's takes over a microsecond).
template <bool TEAM>
struct Exchange {
    uint4* buf;      // [2][EV_WARPS], then [2][EV_CTAS]
    int turn, turn_team, warps, ctas, rank;
    __device__ __forceinline__ void sync() const {
        if (!TEAM) {
            __syncthreads();
        } else {
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
    }
    __device__ __forceinline__ const uint4* give(uint4 x) {
        uint4* b = buf + turn * EV_WARPS;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = x;
        __syncthreads();
        return b;
    }
    // the CTA's number, the same in every warp, to all CTAs
    __device__ __forceinline__ const uint4* give_team(uint4 x) {
        uint4* b = buf + 2 * EV_WARPS + turn_team * EV_CTAS;
        turn_team ^= 1;
        if ((int)threadIdx.x < ctas) put_in_cta(in_cta(tq_smem_u32(b + rank), (int)threadIdx.x), x);
        sync();
        return b;
    }
    __device__ __forceinline__ uint4 join(const uint4* b, int n) const {
        const int lane = threadIdx.x & 31;
        const uint4 v = lane < n ? b[lane] : make_uint4(0u, 0u, 0u, 0u);
        return make_uint4(__reduce_add_sync(0xffffffffu, v.x), __reduce_max_sync(0xffffffffu, v.y), __reduce_max_sync(0xffffffffu, v.z), 0u);
    }
    // x: sum; y, z: largest.  `alone`: within this CTA
    __device__ __forceinline__ uint4 trial(uint32_t x, uint32_t y, uint32_t z, bool alone = false) {
        uint4 r = join(give(make_uint4(__reduce_add_sync(0xffffffffu, x), __reduce_max_sync(0xffffffffu, y), __reduce_max_sync(0xffffffffu, z), 0u)), warps);
        if (TEAM && !alone) r = join(give_team(r), ctas);
        return r;
    }
    // sums of two numbers a warp over the warps before this one (x, y) and over all (z, w)
    __device__ __forceinline__ uint4 before(uint32_t x, uint32_t y) {
        const int lane = threadIdx.x & 31;
        auto add = [&](const uint4* b, int n, int me) {
            const uint4 v = lane < n ? b[lane] : make_uint4(0u, 0u, 0u, 0u);
            return make_uint4(__reduce_add_sync(0xffffffffu, lane < me ? v.x : 0u), __reduce_add_sync(0xffffffffu, lane < me ? v.y : 0u),
                              __reduce_add_sync(0xffffffffu, v.x), __reduce_add_sync(0xffffffffu, v.y));
        };
        uint4 r = add(give(make_uint4(x, y, 0u, 0u)), warps, (int)(threadIdx.x >> 5));
        if (TEAM) {
            const uint4 t = add(give_team(make_uint4(r.z, r.w, 0u, 0u)), ctas, rank);
            r = make_uint4(r.x + t.x, r.y + t.y, t.z, t.w);
        }
        return r;
    }
};

// A thread holds EV_KPT slots as keys in registers; a row that is longer than the team holds (LONG) is gone over again for every
// count.  Masses and positions are read again where they are written: they are in the caches.
template <bool TEAM, bool LONG>
__global__ void __maxnreg__(56) tq_pages_evict_kernel(const EvictParams p) {
    constexpr int KPT = EV_KPT;
    __shared__ uint4 s_buf[2 * EV_WARPS + 2 * EV_CTAS];
    __shared__ uint32_t s_some[TEAM ? EV_SOME : 1];        // of a team's first CTA: the keys left for it
    __shared__ uint32_t s_few[EV_FEW], s_count[2];         // the keys left for one warp; their numbers
    __shared__ uint4 s_found;                              // the limit, and how many equal to it are taken
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t below = (1u << lane) - 1u;
    int ctas = 1, rank = 0;
    if (TEAM) {
        asm("mov.u32 %0, %cluster_nctarank;" : "=r"(ctas));
        asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    }
    const int row = blockIdx.x / ctas, b = row / p.g.H;
    Exchange<TEAM> team{s_buf, 0, 0, warps, ctas, rank};
    if (threadIdx.x < 2) s_count[threadIdx.x] = 0;
    if (TEAM) team.sync();                             // the others have begun: their shared memory may be written
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int n = seq_len(p.q, b, p.status), m = min(n, p.budget);
    const int held = p.held[b], seen = p.seen[b], late = seen + n - held - p.recent;
    const float* mass = p.mass + row * p.stride;
    const int32_t* positions = p.positions + row * p.stride;
    float* out_mass = p.out_mass + row * p.out_stride;
    int32_t* out_positions = p.out_positions + row * p.out_stride;
    const int64_t first = (int64_t)row * p.list;
    int32_t *dst = p.dst + first, *src = p.src + first, *src_positions = p.src_positions + first;
    float* src_mass = p.src_mass + first;
    const int span = ctas * warps * 32 * KPT, rounds = LONG ? (n + span - 1) / span : 1;

    uint32_t key[KPT];                 // 0: not in the cache
    uint32_t guard = 0;                // bit i: slot i of this thread is protected
    auto first_slot = [&](int r) { return r * span + (rank * warps + w) * 32 * KPT + lane; };
    auto position = [&](int t) { return t < held ? positions[t] : seen + t - held; };
    auto load = [&](int r) {
        const int t0 = first_slot(r);
        float x[KPT];
        int pos[KPT];
#pragma unroll
        for (int i = 0; i < KPT; ++i) x[i] = t0 + i * 32 < n ? mass[t0 + i * 32] : 0.f;
#pragma unroll
        for (int i = 0; i < KPT; ++i) pos[i] = t0 + i * 32 < n ? position(t0 + i * 32) : 0;
        guard = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const bool there = t0 + i * 32 < n;
            key[i] = there ? key_of(x[i]) : 0u;
            guard |= (uint32_t)(there && pos[i] >= late) << i;
        }
    };
    load(0);

    // protected tokens first; the rest by key, or the protected by key where they alone exceed the budget
    const bool trims = n > m;
    bool all_guarded = false;          // the candidates are the protected tokens
    uint32_t limit = 0u;               // the k-th largest key of the candidates
    int equal_taken = 0;               // how many of the keys equal to it are taken, lowest slots first
    auto among = [&](int i) { return ((guard >> i) & 1u) == (uint32_t)all_guarded; };
    auto drop = [&]() {                // keys of others than candidates are 0, and no trial value is
#pragma unroll
        for (int i = 0; i < KPT; ++i)
            if (!among(i)) key[i] = 0u;
    };
    if (trims) {
        int guarded = 0;
        uint32_t low = 0u, high = 0u;                      // of the candidates' keys: the largest complement, the largest
        auto ends_of = [&]() {
#pragma unroll
            for (int i = 0; i < KPT; ++i)
                if (key[i] != 0u && among(i)) low = max(low, ~key[i]), high = max(high, key[i]);
        };
        for (int r = 0; r < rounds; ++r) {
            if (LONG && r > 0) load(r);
            guarded += __popc(guard);
            ends_of();
        }
        uint4 ends = team.trial((uint32_t)guarded, low, high);
        guarded = (int)ends.x;
        if (guarded >= m) {                                // the protected ones alone are too many
            all_guarded = true;
            low = high = 0u;
            for (int r = 0; r < rounds; ++r) {
                if (LONG) load(r);
                ends_of();
            }
            ends = team.trial(0u, low, high);
        }
        const int k = all_guarded ? m : m - guarded;
        drop();
        // the k-th largest lies from lo to hi, both keys of the row: `reach` keys are >= lo, `above` > hi
        uint32_t lo = ~ends.y, hi = ends.z;
        int reach = all_guarded ? guarded : n - guarded, above = 0;
        // a trial: the keys that reach it, the largest below it, the complement of the least that reaches it
        auto count = [&](uint32_t trial, int& c, uint32_t& under, uint32_t& over) {
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                const bool there = key[i] >= trial;
                c += there;
                if (there) over = max(over, ~key[i]);
                else under = max(under, key[i]);
            }
        };
        const int few = TEAM ? (int)blockDim.x * KPT : EV_FEW;
        while (k > 0 && lo < hi && reach != k && reach - above > few) {
            const uint32_t trial = lo + (hi - lo) / 2 + 1;
            int c = 0;
            uint32_t under = 0u, over = 0u;
            for (int r = 0; r < rounds; ++r) {
                if (LONG) {
                    load(r);
                    drop();
                }
                count(trial, c, under, over);
            }
            const uint4 got = team.trial((uint32_t)c, under, over);
            if ((int)got.x >= k) lo = ~got.z, reach = (int)got.x;
            else hi = got.y, above = (int)got.x;
        }
        if (k == 0) {                                      // nothing but the protected ones
            limit = 0xffffffffu;
        } else if (reach == k || lo == hi) {
            limit = lo;
            equal_taken = reach == k ? 0x7fffffff : k - above;
        } else {
            // the keys from lo to hi go to fewer hands: those of a team to its first CTA, whose go on, and those to one warp
            auto collect = [&](uint32_t* list, uint32_t* number, int most) {
                const uint32_t count_at = in_cta(tq_smem_u32(number), 0), list_at = in_cta(tq_smem_u32(list), 0);
#pragma unroll
                for (int i = 0; i < KPT; ++i)
                    if (key[i] >= lo && key[i] <= hi) {
                        uint32_t at;
                        asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(count_at) : "memory");
                        if (at < (uint32_t)most) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(list_at + at * 4), "r"(key[i]) : "memory");
                    }
            };
            if (TEAM) {
                for (int r = 0; r < rounds; ++r) {
                    if (LONG) {
                        load(r);
                        drop();
                    }
                    collect(s_some, s_count, EV_SOME);
                }
                team.sync();
            }
            bool settled = false;
            if (!TEAM || rank == 0) {
                uint32_t held_keys[KPT];                   // a team's first CTA: its own keys make room for those left
                if (TEAM) {
#pragma unroll
                    for (int i = 0; i < KPT; ++i) {
                        held_keys[i] = key[i];
                        const int j = i * (int)blockDim.x + (int)threadIdx.x;
                        key[i] = j < (int)s_count[0] ? s_some[j] : 0u;
                    }
                    // of them: `above` lie over hi
                    const int want = k - above;
                    int there = reach - above, over_hi = 0;
                    while (lo < hi && there != want && there - over_hi > EV_FEW) {
                        const uint32_t trial = lo + (hi - lo) / 2 + 1;
                        int c = 0;
                        uint32_t under = 0u, over = 0u;
                        count(trial, c, under, over);
                        const uint4 got = team.trial((uint32_t)c, under, over, true);
                        if ((int)got.x >= want) lo = ~got.z, there = (int)got.x;
                        else hi = got.y, over_hi = (int)got.x;
                    }
                    reach = there + above;
                    above += over_hi;
                    settled = lo == hi || reach == k;
                }
                if (!settled) {
                    collect(s_few, s_count + 1, EV_FEW);
                    __syncthreads();
                }
                if (TEAM) {
#pragma unroll
                    for (int i = 0; i < KPT; ++i) key[i] = held_keys[i];
                }
            }
            if (rank == 0 && w == 0) {
                uint32_t mine[EV_FEW / 32];
#pragma unroll
                for (int i = 0; i < EV_FEW / 32; ++i) mine[i] = !settled && i * 32 + lane < (int)s_count[1] ? s_few[i * 32 + lane] : 0u;
                const int want = k - above;
                int there = reach - above, over = 0;       // of the few: >= lo, > hi
                while (lo < hi && there != want) {
                    const uint32_t trial = lo + (hi - lo) / 2 + 1;
                    int c = 0;
                    uint32_t under = 0u, least = 0u;
#pragma unroll
                    for (int i = 0; i < EV_FEW / 32; ++i) {
                        c += mine[i] >= trial;
                        if (mine[i] >= trial) least = max(least, ~mine[i]);
                        else under = max(under, mine[i]);
                    }
                    c = (int)__reduce_add_sync(0xffffffffu, c);
                    if (c >= want) lo = ~__reduce_max_sync(0xffffffffu, least), there = c;
                    else hi = __reduce_max_sync(0xffffffffu, under), over = c;
                }
                const uint4 found = make_uint4(lo, there == want ? 0x7fffffffu : (uint32_t)(want - over), 0u, 0u);
                if (lane < ctas) put_in_cta(in_cta(tq_smem_u32(&s_found), lane), found);
            }
            team.sync();
            limit = s_found.x;
            equal_taken = (int)s_found.y;
        }
    }

    // the lists, in ascending order: holes before m, movers behind it
    int equals = 0, holes = 0, movers = 0;                 // of the slots before this round
    for (int r = 0; r < rounds; ++r) {
        if (LONG) {
            load(r);
            if (trims) drop();
        }
        const int t0 = first_slot(r);
        int rank_eq = 0;
        if (trims && equal_taken != 0x7fffffff) {          // ranks of the keys equal to the limit, where not all are taken
            int mine = 0;
#pragma unroll
            for (int i = 0; i < KPT; ++i) mine += __popc(__ballot_sync(0xffffffffu, key[i] != 0u && key[i] == limit));
            const uint4 at = team.before((uint32_t)mine, 0u);
            rank_eq = equals + (int)at.x;
            equals += (int)at.z;
        }
        uint32_t kept = 0;                                 // bit i: slot i of this thread stays in the cache
        int my_holes = 0, my_movers = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            bool stays = t < n;
            if (trims) {
                const uint32_t eq = __ballot_sync(0xffffffffu, key[i] != 0u && key[i] == limit);
                stays = stays && (among(i) ? key[i] > limit || (key[i] == limit && rank_eq + __popc(eq & below) < equal_taken) : !all_guarded);
                rank_eq += __popc(eq);
            }
            my_holes += __popc(__ballot_sync(0xffffffffu, t < m && !stays));
            my_movers += __popc(__ballot_sync(0xffffffffu, t >= m && stays));
            kept |= (uint32_t)stays << i;
        }
        float x[KPT];
        int pos[KPT];
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            if ((kept >> i) & 1) x[i] = mass[t], pos[i] = position(t);
        }
        int hole_at = 0, mover_at = 0;
        if (trims) {
            const uint4 at = team.before((uint32_t)my_holes, (uint32_t)my_movers);
            hole_at = holes + (int)at.x, mover_at = movers + (int)at.y;
            holes += (int)at.z, movers += (int)at.w;
        }
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int t = t0 + i * 32;
            const bool stays = (kept >> i) & 1;
            if (trims) {
                const uint32_t hole = __ballot_sync(0xffffffffu, t < m && !stays);
                if (t < m && !stays) dst[hole_at + __popc(hole & below)] = t;
                hole_at += __popc(hole);
            }
            if (t < m && stays) out_mass[t] = x[i], out_positions[t] = pos[i];
            if (trims) {
                const uint32_t mover = __ballot_sync(0xffffffffu, t >= m && stays);
                const int at = mover_at + __popc(mover & below);
                if (t >= m && stays) src[at] = t, src_mass[at] = x[i], src_positions[at] = pos[i];
                mover_at += __popc(mover);
            }
        }
    }
    // in place: nothing is cleared before it has been read (in a row that the team holds, before the last exchange)
    if (LONG) team.sync();
    for (int64_t t = m + rank * (int)blockDim.x + (int)threadIdx.x; t < p.out_stride; t += ctas * blockDim.x) {
        out_mass[t] = 0.f;
        out_positions[t] = -1;
    }
    if (rank == 0 && threadIdx.x == 0) p.count[row] = holes;
}

// The moves of all (sequence, kv head) rows: a group of D/8 lanes copies a key row and a value row.  Bound by HBM: 3500 rows of each of
// 32 heads of 128, 115 MB: 20 us (two rows a group at a time 21.5, four 25: more groups beat more loads of one).  The list is read
// beside its length: 0.6 us of a call's chain.
template <int D>
__global__ void __launch_bounds__(256) tq_pages_move_kernel(const EvictParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int LPR = D / 8, PER = 256 / LPR;
    const int row = blockIdx.x, b = row / p.g.H, h = row % p.g.H;
    const int32_t* table = p.q.table + (int64_t)b * p.q.table_stride;
    const int64_t first = (int64_t)row * p.list, o = (threadIdx.x % LPR) * 16 + h * p.g.sh;
    const bool leads = threadIdx.x % LPR == 0;             // of the group: the ledger's entry is its
    int j = blockIdx.y * PER + threadIdx.x / LPR, from, to, position;
    float mass;
    auto look_up = [&]() {
        from = p.src[first + j], to = p.dst[first + j];
        if (leads) mass = p.src_mass[first + j], position = p.src_positions[first + j];
    };
    if (j < p.list) look_up();                             // beside the count, which says whether it is one
    const int count = p.count[row];
    while (j < count) {
        const int fp = p.g.by_page.quotient(from), tp = p.g.by_page.quotient(to), eb = table[fp], tb = table[tp];
        if (leads) p.out_mass[row * p.out_stride + to] = mass, p.out_positions[row * p.out_stride + to] = position;
        if ((uint32_t)eb < (uint64_t)p.g.num_blocks && (uint32_t)tb < (uint64_t)p.g.num_blocks) {
            const int64_t s = eb * p.g.sb + (int64_t)(from - fp * p.g.page) * p.g.st + o;
            const int64_t d = tb * p.g.sb + (int64_t)(to - tp * p.g.page) * p.g.st + o;
            const uint4 k = *reinterpret_cast<const uint4*>(p.g.k + s), v = *reinterpret_cast<const uint4*>(p.g.v + s);
            *reinterpret_cast<uint4*>(p.g.k + d) = k;
            *reinterpret_cast<uint4*>(p.g.v + d) = v;
        } else {
            atomicCAS(p.status, 0, (int)TQ_ERR_RANGE);
        }
        j += gridDim.y * PER;
        if (j < count) look_up();
    }
    if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0) {   // here, not in the first launch: other heads of the sequence read them there
        const int n = seq_len(p.q, b, p.status), held = p.held[b], seen = p.seen[b];
        p.new_lens[b] = min(n, p.budget);
        p.out_seen[b] = seen + n - held;
        p.out_held[b] = min(n, p.budget);
    }
}

int evict_list(const tq_pages_batch* q, int budget) {      // moves of a row at most
    const int behind = q->max_seq_len - budget;
    return behind <= 0 ? 0 : behind < budget ? behind : budget;
}
// Two arrays that are neither the same nor apart: rows of one would be written before the other's are read.
bool half_over(const void* a, int64_t a_words, const void* b, int64_t b_words) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return !(x == y && a_words == b_words) && x < y + b_words * 4 && y < x + a_words * 4;
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
    *out = rows * 4 + rows * evict_list(batch, budget) * 16;
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
    const int64_t rows = (int64_t)batch->batch * pages->num_kv_heads, words = rows * ledger->max_tokens, out_words = rows * out->max_tokens;
    if (half_over(ledger->mass, words, out->mass, out_words) || half_over(ledger->positions, words, out->positions, out_words) ||
        half_over(ledger->held, batch->batch, out->held, batch->batch) || half_over(ledger->seen, batch->batch, out->seen, batch->batch))
        return TQ_ERR_SHAPE;
    if (scratch_bytes < need) return TQ_ERR_WORKSPACE;
    if ((uintptr_t)scratch & 15) return TQ_ERR_ALIGN;
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
    p.src_positions = p.src + rows * p.list;
    p.src_mass = reinterpret_cast<float*>(p.src_positions + rows * p.list);
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    tq_note_launch(st, TQ_LAUNCH_LENGTHS);     // writes rows that a store may read next, and lengths that a decode may
    // as many CTAs a row as it takes to hold its keys in registers, up to eight; no more warps than hold them
    const int n = batch->max_seq_len, cta = EV_WARPS * 32 * EV_KPT;
    const int ctas = n <= cta ? 1 : n <= 2 * cta ? 2 : n <= 4 * cta ? 4 : EV_CTAS;
    const int each = (n + ctas - 1) / ctas, threads = each >= cta ? EV_WARPS * 32 : (each + 32 * EV_KPT - 1) / (32 * EV_KPT) * 32;
    if (rows * ctas >= ((int64_t)1 << 31)) return TQ_ERR_SHAPE;
    const dim3 teams((unsigned)(rows * ctas));
    const int rc2 = ctas == 1 ? launch_behind(tq_pages_evict_kernel<false, false>, teams, threads, 0, st, p)
                    : n <= ctas * cta ? launch_behind_in_clusters(tq_pages_evict_kernel<true, false>, teams, threads, ctas, st, p)
                                      : launch_behind_in_clusters(tq_pages_evict_kernel<true, true>, teams, threads, ctas, st, p);
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
