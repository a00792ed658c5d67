// Beam search's selection: from the logits of every beam and the beams' scores to the next beams.
//
//   total(g, b, v) = score(g, b) + (x(b, v) - m(b)) - log sum_u exp(x(b, u) - m(b)),   m(b) the largest logit of the row
//
// A group's candidates are ordered by total, descending, and by (b, v) where totals are equal.  The first ``beams`` of them whose
// token is no stop token go on; those among the first ``beams`` of all whose token is one have ended.  NaN counts as -infinity,
// +infinity as the largest finite number; a candidate at -infinity is none, so masked tokens and beams at -infinity never win.
//
// Two kernels.  The scan reads every logit once, a warp to a tile of 1,024, and leaves a tile's largest logit and its sum of
// exponentials.  The merge, a block per group, knows from these each row's sum and each tile's largest total.  The ``beams``-th
// largest of the tiles' totals (not counting tiles whose largest logit is a stop token's) is a bound that no chosen candidate lies
// below, and only tiles that reach it hold any: about ``beams`` tiles of a whole group.  Those are read again, out of L2, and what
// lies above the bound is ranked by counting.  So the pass over the vocabulary selects nothing; it is a maximum and a sum.
//
// Where so many candidates are equal that they overflow the room (tokens masked with the lowest number, constant rows), the tiles
// are taken one by one in the order of (b, v), each cut down to the best so far: an equal total that comes later loses, so that
// tiles which only reach the bound are passed over from then on.
//
// Totals, sums and the order are in 64 bits, a sum good to 5e-11: beams compete by sums over a whole vocabulary, and at 32 bits the
// order of two candidates of different rows would depend on how the sums were split.  Scores come and go in 32 or in 64 bits: a search
// that hands them over in 32 rounds the whole sum at every step, and after 1,500 tokens near -3.7 each was off by 0.016.
#include "common.cuh"

namespace {
constexpr int BEAMS_MAX = 32;        // a group's beams: one bit of a warp's word each
constexpr int STOPS_MAX = 16;
constexpr int TILE = 1024;           // logits that a warp takes
constexpr int LANE = TILE / 32;
constexpr int SCAN_WARPS = 2;        // a scan block's; warps that share nothing but the table, so small blocks leave no SM waiting
constexpr int MT = 1024;             // threads of a merge block
constexpr int MW = MT / 32;
constexpr int SIDES = MT / 256;      // tiles that are read again side by side
constexpr int TILES = 512;           // tiles of a group that may reach the bound
constexpr int ROOM = 1536;           // candidates above it; more than a tile and all that is kept of the ones before
// Tiles of a group whose totals are kept in shared memory: what its 48 KB leave, 25 rows of 151,936 logits.  The others' parts are read again
// from L2: 16 us for 26 such rows, 17 to 18 for 32, wherever the best scores are.
constexpr int KEYS = 3840;
constexpr int AHEAD = 2;             // tiles that each side has on the way at a time
// Tiles of a row, of 32 each, whose parts a warp has on the way at a time; rows of up to 5 * 32 * 1,024 = 163,840 logits are read once (24 of
// them 15.9 us, 17.1 for 24 of 164,000).
constexpr int HELD = 5;
constexpr float BIG = 3.402823466e38f;
constexpr float PLAIN = 600.f;       // |largest logit| of a tile up to which its exponentials are summed as they are
constexpr float LEAST = -690.f;      // what lies below counts as this: e^-690, next to nothing beside e^-600
constexpr unsigned KEY_NONE = 0x007FFFFFu;      // the key of -infinity: the least key of all

__device__ __forceinline__ unsigned order_key(float x) {
    if (x == 0.f) x = 0.f;      // -0 counts as +0
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(double x) {
    if (x == 0.0) x = 0.0;
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double total_of(unsigned long long key) {
    return __longlong_as_double((long long)((key >> 63) ? key & 0x7FFFFFFFFFFFFFFFull : ~key));
}
// a total's 32-bit key: keeps the order, not strictly
__device__ __forceinline__ unsigned short_key(double total) { return order_key(__double2float_rd(total)); }

// 2^(j/16)
__constant__ double pow16[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484,
                                 1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993, 1.5422108254079407,
                                 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// sum + exp(x), -690 <= x <= 690 (a larger one gives anything), relative error below 5e-11; after Tang, "Table-driven implementation of
// the exponential function in IEEE floating-point arithmetic", 1989: x = (16 n + j) ln 2 / 16 + r with |r| <= ln 2 / 32, exp(x) =
// 2^n 2^(j/16) exp(r), and exp(r) - 1 - r - ... - r^4/24 is at most r^5 / 120 = 4e-11.  k = 16 n + j is rounded by adding 1.5 * 2^52, whose
// last bits are then k; ``table`` holds 2^(j/16) with j taken off bit 16 on of its high word, so that adding k << 16 there multiplies by
// 2^n.  Eight operations of 64 bits: 64 rows of 151,936 logits take 11.0 us, 15.8 with exp(), 7.2 with no exponential.  (With r and the
// polynomial in 32 bits, two values at a time, 9.5, but a sum in which one term prevails is then good to 1e-8 only.)
__device__ __forceinline__ double add_exp(double sum, double x, const double* __restrict__ table) {
    const double t = fma(x, 23.083120654223414, 6755399441055744.0);
    const int k = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -0.04332169878499658, x);
    const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0);
    const double f = table[k & 15];
    return fma(__hiloint2double(__double2hiint(f) + (int)((unsigned)k << 16), __double2loint(f)), p, sum);
}

struct __align__(16) Part {              // of a tile
    double sum;          // of exp(x - ref)
    float top;           // the largest logit; -infinity: none, and the rest is not written
    float ref;           // 0, or ``top`` where the exponentials would leave the range of 64 bits
};

struct ScanArgs {
    const float* logits;
    long long ld;
    int V, tiles;
    const void* scores;  // float32 or float64: the kernels' S
    Part* part;          // [rows, tiles]
};

// A lane's entry e of the tile that begins at ``at``.  VEC: four neighbouring ones at a time (rows that start at 16 bytes).
template <bool VEC>
__device__ __forceinline__ int place_of(int at, int e, int lane) {
    return VEC ? at + ((e >> 2) * 32 + lane) * 4 + (e & 3) : at + e * 32 + lane;
}

template <bool VEC>
__device__ __forceinline__ void load_tile(float (&v)[LANE], const float* x, int at, int V, int lane) {
    if (VEC && at + TILE <= V) {
#pragma unroll
        for (int e = 0; e < LANE; e += 4) {
            const float4 q = *reinterpret_cast<const float4*>(x + place_of<true>(at, e, lane));
            v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < LANE; ++e) {
            const int i = place_of<VEC>(at, e, lane);
            v[e] = i < V ? x[i] : -INFINITY;
        }
    }
}

// A lane's entries, and so the order of a row's sum, depend on their places alone: equal rows have equal sums.
template <bool VEC, typename S>
__global__ void __launch_bounds__(SCAN_WARPS * 32, 16) beam_scan_kernel(ScanArgs a) {
    ti_pdl_trigger();
    __shared__ double table[16];
    const int lane = threadIdx.x & 31, tile = blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5), row = blockIdx.y;
    if (threadIdx.x < 16)
        table[threadIdx.x] = __hiloint2double(__double2hiint(pow16[threadIdx.x]) - ((int)threadIdx.x << 16), __double2loint(pow16[threadIdx.x]));
    __syncthreads();
    ti_pdl_sync();
    const S* scores = static_cast<const S*>(ti_dependent(a.scores));
    const float* x = ti_dependent(a.logits) + (size_t)row * a.ld;
    if (tile >= a.tiles || !(scores[row] > (S)-INFINITY)) return;      // (the merge leaves such a row out as well)
    float v[LANE];
    load_tile<VEC>(v, x, tile * TILE, a.V, lane);
    float top = -INFINITY;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int e = 0; e < LANE; ++e) {
        top = fmaxf(top, v[e]);              // (a NaN is passed over, and counts as LEAST below)
        s[e & 3] = add_exp(s[e & 3], (double)fmaxf(v[e], LEAST), table);
    }
    top = warp_max(fminf(top, BIG));
    const bool plain = fabsf(top) <= PLAIN;
    if (!plain && top > -INFINITY) {
        s[0] = s[1] = s[2] = s[3] = 0.0;
#pragma unroll
        for (int e = 0; e < LANE; ++e)
            if (v[e] > -INFINITY) s[e & 3] = add_exp(s[e & 3], fmax((double)fminf(v[e], BIG) - (double)top, (double)LEAST), table);
    }
    double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) a.part[(size_t)row * a.tiles + tile] = Part{sum, top, plain ? 0.f : top};
}

// A value at or below the k-th largest (k <= 32) of the block's keys (one per thread, in shared memory), with few keys more above it
// than k; by one warp.  Of two keys the larger one stands for both, and every lane holds MW / 2 of those; at least 32 lie at or above
// the least of the lanes' largest ones: there the bisection begins, and it is mostly done after a step or two.
__device__ __forceinline__ unsigned bound_of(const unsigned* __restrict__ keys, int k) {
    const int lane = threadIdx.x & 31;
    unsigned mine[MW / 2], first = 0u;
#pragma unroll
    for (int i = 0; i < MW / 2; ++i) {
        mine[i] = max(keys[i * 32 + lane], keys[(i + MW / 2) * 32 + lane]);
        first = max(first, mine[i]);
    }
    unsigned lo = __reduce_min_sync(0xffffffffu, first), hi = __reduce_max_sync(0xffffffffu, first);
    const int enough = k + (k >> 1) + 2;
    auto above = [&](unsigned bound) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < MW / 2; ++i) n += mine[i] >= bound;
        return __reduce_add_sync(0xffffffffu, n);
    };
    if (above(max(lo, KEY_NONE + 1)) <= enough) return lo;
#pragma unroll 1
    while (lo < hi) {
        const unsigned mid = lo + ((hi - lo) >> 1) + 1;
        const int n = above(mid);
        if (n >= k) {
            lo = mid;
            if (n <= enough) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

struct MergeArgs {
    const float* logits;
    long long ld;
    const void* scores;      // [groups, held]
    const Part* part;
    const int* stops;
    int held, beams, n_stops, tiles, V, ending;
    void* out_score;         // [groups, beams], by place, of the type of ``scores`` as ``end_score`` is
    int* out_parent;
    int* out_token;
    void* end_score;         // [groups, beams], by rank
    int* end_parent;
    int* end_token;
};

// What a block of the merge spends is latency: instructions that a block runs once come from L2 as its data do, so the code is kept
// in loops, and what is rare is out of the way.  Behind the scan it takes 5 us for one row of 151,936 as for a group of four, 10
// for 24 rows of 123,373 at odd addresses (12 with 512 threads, 19 with 256; one row 0.5 us less with 512).
template <bool VEC, typename S>
__global__ void __launch_bounds__(MT) beam_merge_kernel(MergeArgs a) {
    ti_pdl_trigger();
    __shared__ unsigned tile_key[KEYS];                              // a tile's top logit, then its largest total's key
    __shared__ unsigned keys[MT];
    __shared__ unsigned stop_tile[KEYS / 32];                        // a bit per tile: its top logit is a stop token's
    __shared__ unsigned long long found_key[ROOM], found_at[ROOM];   // a total's key; beam << 32 | token, with the top bit for a stop token
    __shared__ int tile_list[TILES];                                 // beam << 24 | tile
    __shared__ double row_add[BEAMS_MAX], row_ref[BEAMS_MAX];        // a total is row_add + (x - row_ref); row_add -infinity: no beam
    __shared__ float row_cut[BEAMS_MAX];                             // logits below it do not reach the bound
    __shared__ S next_score[BEAMS_MAX];
    __shared__ int next_parent[BEAMS_MAX], next_token[BEAMS_MAX], free_place[BEAMS_MAX];
    __shared__ int stops[STOPS_MAX];
    __shared__ int n_tiles, n_found, s_first;
    __shared__ unsigned s_bound;
    __shared__ unsigned long long s_last;
    constexpr unsigned long long STOP = 1ull << 63;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.x, all = a.held * a.tiles;
    for (int i = tid; i < KEYS / 32; i += MT) stop_tile[i] = 0u;
    if (tid < BEAMS_MAX) {
        next_parent[tid] = -1;
        row_add[tid] = -INFINITY;
    }
    if (tid == 0) n_tiles = n_found = 0;
    ti_pdl_sync();
    const S* scores = static_cast<const S*>(ti_dependent(a.scores)) + (size_t)g * a.held;
    S *out_score = static_cast<S*>(a.out_score), *end_score = static_cast<S*>(a.end_score);
    const float* logits = ti_dependent(a.logits) + (size_t)g * a.held * a.ld;
    const Part* part = ti_dependent(a.part) + (size_t)g * all;
    const int* stop_ids = ti_dependent(a.stops);
    const size_t o = (size_t)g * a.beams;
    if (tid < a.n_stops) stops[tid] = stop_ids[tid];
    if (tid < a.beams) {
        end_score[o + tid] = (S)-INFINITY;
        a.end_parent[o + tid] = -1;
        a.end_token[o + tid] = -1;
    }
    __syncthreads();
    auto is_stop = [&](int token) {
        bool stop = false;
#pragma unroll 1
        for (int s = 0; s < a.n_stops; ++s) stop |= stops[s] == token;
        return stop;
    };
    // A tile whose top logit is a stop token's says nothing about the others' totals.
#pragma unroll 1
    for (int i = MT - 1 - tid; i < a.held * a.n_stops; i += MT) {
        const int b = i / a.n_stops, id = stops[i % a.n_stops], at = b * a.tiles + id / TILE;
        if (id < 0 || id >= a.V || at >= KEYS) continue;
        const float w = logits[(size_t)b * a.ld + id], top = part[at].top;
        if (fminf(w, BIG) == top) atomicOr(&stop_tile[at >> 5], 1u << (at & 31));
    }
    // Each row's sum, by a warp, and from it the keys of its tiles' largest totals: 0 where a tile has no candidate.
#pragma unroll 1
    for (int b = warp; b < a.held; b += MW) {
        const Part* p = part + (size_t)b * a.tiles;
        const S score = scores[b];
        bool some = false, shifted = false;
        double sum = 0.0;
        Part q[HELD];
#pragma unroll 1
        for (int t0 = 0; t0 < a.tiles; t0 += HELD * 32) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) q[j] = t0 + j * 32 + lane < a.tiles ? p[t0 + j * 32 + lane] : Part{0.0, -INFINITY, 0.f};
#pragma unroll
            for (int j = 0; j < HELD; ++j)
                if (q[j].top > -INFINITY) {
                    some = true;
                    shifted |= q[j].ref != 0.f;
                    sum += q[j].sum;
                }
        }
        const bool there = score > (S)-INFINITY && __any_sync(0xffffffffu, some);      // (nothing was written for a row without a beam)
        float m = 0.f;
        if (there && __any_sync(0xffffffffu, shifted)) {
            // tiles that were taken against another reference than 0: all against the largest of them
            m = -INFINITY;
#pragma unroll 1
            for (int t = lane; t < a.tiles; t += 32)
                if (p[t].top > -INFINITY) m = fmaxf(m, p[t].ref);
            m = warp_max(m);
            sum = 0.0;
#pragma unroll 1
            for (int t = lane; t < a.tiles; t += 32)
                if (p[t].top > -INFINITY) sum += p[t].sum * exp((double)p[t].ref - (double)m);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const double add = there ? (double)score - log(sum) : -INFINITY, ref = m;
        if (lane == 0) {
            row_add[b] = add;
            row_ref[b] = ref;
        }
#pragma unroll 1
        for (int t0 = 0; t0 < a.tiles; t0 += HELD * 32) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const int t = t0 + j * 32 + lane, i = b * a.tiles + t;
                if (t >= a.tiles || i >= KEYS) continue;
                const float top = a.tiles > HELD * 32 ? p[t].top : q[j].top;
                tile_key[i] = there && top > -INFINITY ? short_key(add + ((double)top - ref)) : 0u;
            }
        }
    }
    __syncthreads();
    // (Tiles behind the shared ones are read again each time, and count for the bound only where they hold no stop token at all.)
    auto key_behind = [&](int i) {
        const int b = i / a.tiles;
        const float top = part[i].top;
        return row_add[b] > -INFINITY && top > -INFINITY ? short_key(row_add[b] + ((double)top - row_ref[b])) : 0u;
    };
    unsigned mine = KEY_NONE;
    const int shared = min(all, KEYS);
#pragma unroll 2
    for (int i = tid; i < shared; i += MT)
        if (!((stop_tile[i >> 5] >> (i & 31)) & 1u)) mine = max(mine, tile_key[i]);
#pragma unroll 1
    for (int i = KEYS + tid; i < all; i += MT) {
        bool stop = false;
#pragma unroll 1
        for (int s = 0; s < a.n_stops; ++s) stop |= stops[s] / TILE == i % a.tiles;
        if (!stop) mine = max(mine, key_behind(i));
    }
    keys[tid] = mine;
    __syncthreads();
    // the bound, and below which logit a row's entries cannot reach it: a little lower, for the roundings of the two forms
    auto cut_rows = [&](unsigned b) {
        const unsigned u = (b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b;
        if (lane == 0) s_bound = b;
        if (lane < a.held) {
            const double t = (double)__uint_as_float(u), add = row_add[lane], ref = row_ref[lane];
            const double cut = ((t - add) + ref) - 1e-14 * (fabs(t) + fabs(add) + fabs(ref));
            row_cut[lane] = b <= KEY_NONE || cut != cut ? -INFINITY : __double2float_rd(cut);
        }
    };
    if (warp == 0) cut_rows(bound_of(keys, a.beams));
    __syncthreads();
    const unsigned bound = s_bound;
    auto list = [&](int i) {
        const int to = atomicAdd(&n_tiles, 1);
        if (to < TILES) tile_list[to] = (i / a.tiles) << 24 | (i % a.tiles);
    };
#pragma unroll 2
    for (int i = tid; i < shared; i += MT)
        if (tile_key[i] >= bound) list(i);
#pragma unroll 1
    for (int i = KEYS + tid; i < all; i += MT)
        if (key_behind(i) >= bound) list(i);
    __syncthreads();
    // a logit's total, and whether it is a candidate at all
    auto candidate = [&](int b, float w, double& total) {
        if (!(w > -INFINITY)) return false;
        total = row_add[b] + ((double)fminf(w, BIG) - row_ref[b]);
        return total > -INFINITY;
    };
    auto put = [&](int i, double total, int b, int token) {
        found_key[i] = order_key(total);
        found_at[i] = ((unsigned long long)b << 32 | (unsigned)token) | (is_stop(token) ? STOP : 0ull);
    };
    // f(beam, token, logit) for the listed tiles' entries that reach their row's cut
    const int listed = n_tiles;
    auto each = [&](auto&& f) {
#pragma unroll 1
        for (int i0 = tid >> 8; i0 < listed; i0 += SIDES * AHEAD) {      // 256 threads to a tile, four logits each
            const int part_of = tid & 255;
            float v[AHEAD][4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int what = tile_list[min(i0 + SIDES * u, listed - 1)];
                const float* x = logits + (size_t)(what >> 24) * a.ld;
                const int at = (what & 0xFFFFFF) * TILE;
                if (VEC && at + TILE <= a.V) {
                    const float4 q = *reinterpret_cast<const float4*>(x + at + part_of * 4);
                    v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = at + (VEC ? part_of * 4 + e : e * 256 + part_of);
                        v[u][e] = c < a.V ? x[c] : -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (i0 + SIDES * u >= listed) continue;
                const int what = tile_list[i0 + SIDES * u], b = what >> 24, at = (what & 0xFFFFFF) * TILE;
                const float cut = row_cut[b];
                unsigned hits = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) hits |= v[u][e] >= cut ? 1u << e : 0u;          // (a NaN is none)
                while (hits) {
                    const int e = __ffs(hits) - 1;
                    const float w = e < 2 ? (e ? v[u][1] : v[u][0]) : (e == 2 ? v[u][2] : v[u][3]);
                    hits &= hits - 1u;
                    f(b, at + (VEC ? part_of * 4 + e : e * 256 + part_of), w);
                }
            }
        }
    };
    auto gather = [&](int b, int token, float w) {
        const int to = atomicAdd(&n_found, 1);
        if (to < ROOM) {
            found_key[to] = __float_as_uint(w);
            found_at[to] = (unsigned long long)b << 32 | (unsigned)token;
        }
    };
    int n = ROOM + 1;
    if (listed <= TILES) {
        each(gather);
        __syncthreads();
        n = n_found;
        if (n > ROOM) {
            // With fewer tiles than beams there was no bound, and everything lay above it: the threads' largest entries give one.
            mine = KEY_NONE;
            each([&](int b, int token, float w) {
                double total;
                if (candidate(b, w, total) && short_key(total) > mine && !is_stop(token)) mine = short_key(total);
            });
            keys[tid] = mine;
            __syncthreads();
            if (tid == 0) n_found = 0;
            if (warp == 0) cut_rows(bound_of(keys, a.beams));
            __syncthreads();
            each(gather);
            __syncthreads();
            n = n_found;
        }
    }
    // what has rank ``rank`` among all and ``open`` among those that are no stop tokens (whose: beam, token and the stop bit)
    auto settle = [&](unsigned long long key, unsigned long long whose, int rank, int open) {
        const S total = (S)total_of(key);
        if (whose < STOP) {
            if (open < a.beams) {
                next_score[open] = total;
                next_parent[open] = (int)(whose >> 32);
                next_token[open] = (int)whose;
            }
        } else if (a.ending && rank < a.beams) {
            end_score[o + rank] = total;
            a.end_parent[o + rank] = (int)((whose & ~STOP) >> 32);
            a.end_token[o + rank] = (int)whose;
        }
    };
    if (n <= 32) {
        // nearly always: an entry to a lane of one warp, which has all of the rest to itself
        if (warp != 0) return;
        unsigned long long key = 0ull, whose = ~0ull;            // (the key of a number is never 0)
        if (lane < n) {
            const int b = (int)(found_at[lane] >> 32), token = (int)found_at[lane];
            double total;
            if (candidate(b, __uint_as_float((unsigned)found_key[lane]), total)) {
                key = order_key(total);
                whose = found_at[lane] | (is_stop(token) ? STOP : 0ull);
            }
        }
        int rank = 0, open = 0;
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const unsigned long long k2 = __shfl_sync(0xffffffffu, key, j), w2 = __shfl_sync(0xffffffffu, whose, j);
            const bool before = (k2 > key) | ((k2 == key) & ((w2 & ~STOP) < (whose & ~STOP)));
            rank += before;
            open += before & (w2 < STOP);
        }
        if (key) settle(key, whose, rank, open);
        __syncwarp();
    } else {
        if (n <= ROOM) {
#pragma unroll 1
            for (int i = tid; i < n; i += MT) {
                const int b = (int)(found_at[i] >> 32);
                double total;
                // (one that is no candidate, a NaN's neighbour at -infinity: behind all others, and told apart below)
                if (candidate(b, __uint_as_float((unsigned)found_key[i]), total)) put(i, total, b, (int)found_at[i]);
                else found_key[i] = 0ull;
            }
            __syncthreads();
        }
        // ranks of entry i among all that were found, and among those that are no stop tokens
        auto rank_of = [&](int i, int& rank, int& open) {
            const unsigned long long key = found_key[i], at = found_at[i] & ~STOP;
            rank = open = 0;
#pragma unroll 2
            for (int j = 0; j < n; ++j) {
                const unsigned long long k2 = found_key[j], w2 = found_at[j];
                const bool before = (k2 > key) | ((k2 == key) & ((w2 & ~STOP) < at));
                rank += before;
                open += before & (w2 < STOP);
            }
        };
        if (n > ROOM) {
            // Equal totals without end: tile by tile in the order of places, keeping what can still be chosen.
            __syncthreads();
            if (tid == 0) {
                n_found = 0;
                s_last = 0ull;               // the key of the beams-th best so far that is no stop token's; 0: fewer than that
            }
            for (int base = 0; base < all; base += MT) {
                const int i = base + tid;
                unsigned long long top_key = 0ull;
                if (i < all && row_add[i / a.tiles] > -INFINITY && part[i].top > -INFINITY)
                    top_key = order_key(row_add[i / a.tiles] + ((double)part[i].top - row_ref[i / a.tiles]));
                int from = 0;
                while (true) {
                    __syncthreads();
                    if (tid == 0) s_first = MT;
                    __syncthreads();
                    // (totals equal to the last one kept come later than it: they lose)
                    if (tid >= from && top_key > s_last) atomicMin(&s_first, tid);
                    __syncthreads();
                    const int first = s_first;
                    if (first == MT) break;
                    from = first + 1;
                    const int b = (base + first) / a.tiles, at = (base + first) % a.tiles * TILE;
                    const unsigned long long last = s_last;
                    for (int c = at + tid; c < min(at + TILE, a.V); c += MT) {
                        double total;
                        if (candidate(b, logits[(size_t)b * a.ld + c], total) && order_key(total) > last) put(atomicAdd(&n_found, 1), total, b, c);
                    }
                    __syncthreads();
                    n = n_found;             // at most a tile and two times BEAMS_MAX
                    unsigned long long key[(ROOM + MT - 1) / MT], whose[(ROOM + MT - 1) / MT];
                    int keep = 0;
                    for (int j = 0; j * MT + tid < n; ++j) {
                        int rank, open;
                        rank_of(j * MT + tid, rank, open);
                        if (found_at[j * MT + tid] < STOP ? open < a.beams : rank < a.beams) {
                            key[keep] = found_key[j * MT + tid];
                            whose[keep++] = found_at[j * MT + tid];
                            if (whose[keep - 1] < STOP && open == a.beams - 1) s_last = key[keep - 1];
                        }
                    }
                    __syncthreads();
                    if (tid == 0) n_found = 0;
                    __syncthreads();
                    for (int j = 0; j < keep; ++j) {
                        const int to = atomicAdd(&n_found, 1);
                        found_key[to] = key[j];
                        found_at[to] = whose[j];
                    }
                }
            }
            __syncthreads();
            n = n_found;
        }
        if (n <= 256) {
            // a warp to an entry, a lane to one it is compared with
#pragma unroll 1
            for (int i = warp; i < n; i += MW) {
                const unsigned long long key = found_key[i], at = found_at[i] & ~STOP;
                int rank = 0, open = 0;
#pragma unroll 1
                for (int j = lane; j - lane < n; j += 32) {
                    const unsigned long long k2 = j < n ? found_key[j] : 0ull, w2 = j < n ? found_at[j] : ~0ull;
                    const bool before = (k2 > key) | ((k2 == key) & ((w2 & ~STOP) < at));
                    rank += __popc(__ballot_sync(0xffffffffu, before));
                    open += __popc(__ballot_sync(0xffffffffu, before & (w2 < STOP)));
                }
                if (lane == 0 && key) settle(key, found_at[i], rank, open);
            }
        } else {
#pragma unroll 1
            for (int i = tid; i < n; i += MT) {
                int rank, open;
                rank_of(i, rank, open);
                if (found_key[i]) settle(found_key[i], found_at[i], rank, open);
            }
        }
        __syncthreads();
        if (warp != 0) return;
    }
    // Placement by one warp, a lane per rank: the first child of a beam stays at its parent's place, the others take the places of
    // the beams without a child, in order.  What is copied is then never what another copy overwrites.
    const int p = next_parent[lane];
    const bool there = p >= 0;
    const unsigned below = (1u << lane) - 1u;
    const unsigned same = __match_any_sync(0xffffffffu, p);
    const bool stays = there && (same & below) == 0u;
    const unsigned kept = __reduce_or_sync(0xffffffffu, stays ? 1u << p : 0u);
    const unsigned goes = __ballot_sync(0xffffffffu, there && !stays);
    if (!((kept >> lane) & 1u)) free_place[__popc(~kept & below)] = lane;
    __syncwarp();
    const int place = stays ? p : there ? free_place[__popc(goes & below)] : -1;
    const unsigned taken = __reduce_or_sync(0xffffffffu, place >= 0 ? 1u << place : 0u);
    if (place >= 0) {
        out_score[o + place] = next_score[lane];
        a.out_parent[o + place] = p;
        a.out_token[o + place] = next_token[lane];
    }
    if (lane < a.beams && !((taken >> lane) & 1u)) {
        out_score[o + lane] = (S)-INFINITY;
        a.out_parent[o + lane] = lane;
        a.out_token[o + lane] = 0;
    }
}
}  // namespace

// scores, and out_scores [2, groups, beams] (the next beams' and the ended ones'): float64 where wide_scores, float32 otherwise; out_places [4, groups, beams]: parents, tokens, and of the
// ended ones parents and tokens; scratch: a Part for every tile of 1,024 logits of every row.
extern "C" int ti_beam_select(const float* logits, long long ld, int groups, int held, int V, const void* scores, int wide_scores,
                              int beams, const int* stops, int n_stops, int ending, void* out_scores, int* out_places, void* scratch,
                              cudaStream_t stream) {
    TI_REQUIRE(groups >= 1 && held >= 1 && V >= 1 && V <= 1 << 30 && ld >= V, "beam select: %d groups of %d rows of %d logits, %lld apart", groups, held, V, ld);
    TI_REQUIRE(beams >= 1 && beams <= BEAMS_MAX && held <= beams, "beam select: %d beams from %d (at most %d, and no fewer than before)",
               beams, held, BEAMS_MAX);
    TI_REQUIRE(n_stops >= 0 && n_stops <= STOPS_MAX && (n_stops == 0 || stops), "beam select: %d stop tokens (at most %d)", n_stops, STOPS_MAX);
    const long long rows = (long long)groups * held;
    TI_REQUIRE(rows <= 65535, "beam select: %lld rows in one call (at most 65535)", rows);
    TI_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "beam select: the scratch must start at 16 bytes");
    const int tiles = (V + TILE - 1) / TILE;
    const bool vec = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    ScanArgs s = {logits, ld, V, tiles, scores, static_cast<Part*>(scratch)};
    const dim3 grid((tiles + SCAN_WARPS - 1) / SCAN_WARPS, (unsigned)rows);
    auto scan = wide_scores ? (vec ? beam_scan_kernel<true, double> : beam_scan_kernel<false, double>)
                            : (vec ? beam_scan_kernel<true, float> : beam_scan_kernel<false, float>);
    TI_CUDA(ti_launch(scan, grid, dim3(SCAN_WARPS * 32), 0, stream, s));
    const size_t n = (size_t)groups * beams;
    void* ended = static_cast<char*>(out_scores) + n * (wide_scores ? 8 : 4);
    MergeArgs m = {logits, ld, scores, s.part, stops, held, beams, n_stops, tiles, V, ending,
                   out_scores, out_places, out_places + n, ended, out_places + 2 * n, out_places + 3 * n};
    auto merge = wide_scores ? (vec ? beam_merge_kernel<true, double> : beam_merge_kernel<false, double>)
                             : (vec ? beam_merge_kernel<true, float> : beam_merge_kernel<false, float>);
    TI_CUDA(ti_launch(merge, dim3(groups), dim3(MT), 0, stream, m));
    return 0;
}
