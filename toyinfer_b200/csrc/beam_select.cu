// Beam search's selection: from the logits of every beam and the beams' scores to the next beams.
//
//   total(g, b, v) = score(g, b) + (x(b, v) - m(b)) - log sum_u exp(x(b, u) - m(b)),   m(b) the largest logit of the row
//
// A group's candidates are ordered by total, descending, and by (b, v) where totals are equal.  The first ``beams`` of them whose
// token is no stop token go on; those among the first ``beams`` of all whose token is one have ended.  NaN counts as -infinity,
// +infinity as the largest finite number; a candidate at -infinity is none, so masked tokens and beams at -infinity never win.
//
// Two kernels.  The scan runs blocks over (chunk, row): a chunk's logits are read once, and from there come its sum of exponentials
// and its best K = beams + stop tokens entries (at most that many of one row can matter: of the first ``beams`` entries that are no
// stop tokens all but the stop tokens before them).  The merge runs a block per group over what the scan left.
//
// The best K of a chunk without sorting it: the K-th largest of the threads' own maxima is a lower bound of the K-th largest
// entry, and few entries lie above it; the threads whose maximum does look at theirs again, and what they find is ranked by
// counting.  The merge finds its ``beams`` in the same way, from the first entries of the chunks' lists.  Where so many entries are
// equal that those above the bound overflow their room, the bound is made exact entry by entry.
//
// Totals, sums and the order are in 64 bits: beams compete by sums over a whole vocabulary, and at 32 bits the order of two
// candidates of different rows would depend on how the sums were split.  exp is 2^(k/16) from a table of sixteen times a polynomial
// of degree four on |r| <= ln 2 / 32 (add_exp below): eight operations of 64 bits, where exp() takes about thirty.
#include "common.cuh"

namespace {
constexpr int BEAMS_MAX = 32;        // a group's beams: one bit of a warp's word each
constexpr int STOPS_MAX = 16;
constexpr int ST = 256;              // threads of a scan block
constexpr int ROOM = 1024;           // entries above the bound that a block can rank
constexpr int MT = 256;              // threads of a merge block
constexpr int HELD = 8;              // entries that a merge thread holds in registers
constexpr float BIG = 3.402823466e38f;
constexpr float PLAIN = 600.f;       // |largest logit| of a chunk up to which its exponentials are summed as they are

__device__ __forceinline__ unsigned order_key(float x) {
    if (x == 0.f) x = 0.f;      // -0 counts as +0
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr unsigned KEY_NONE = 0x007FFFFFu;      // the key of -infinity: the least key of all

// 2^(j/16)
__constant__ double pow16[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// sum + exp(x), x <= 690 (larger ones give anything), relative error below 5e-11; after Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic", 1989.  x = (16 n + j) ln 2 / 16 + r: k = 16 n + j is
// rounded by adding 1.5 * 2^52, whose last bits are then k; ``table`` holds 2^(j/16) with j taken off bit 16 on of its high word, so
// that adding k << 16 there multiplies by 2^n.  exp(r) - 1 - r - ... - r^4/24 is at most r^5 / 120 = 4e-11.
__device__ __forceinline__ double add_exp(double sum, float x, const double* __restrict__ table) {
    const double xd = (double)fmaxf(x, -690.f);          // (NaN and -infinity: next to nothing)
    const double t = fma(xd, 23.083120654223414, 6755399441055744.0);
    const int k = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -0.04332169878499658, xd);
    const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0);
    const double f = table[k & 15];
    return fma(__hiloint2double(__double2hiint(f) + (int)((unsigned)k << 16), __double2loint(f)), p, sum);
}

// A value at or below the k-th largest (k <= 64) of the block's keys (one per thread, in shared memory), with few keys more above it
// than k; by one warp.  Every lane holds THREADS / 32 of the keys, so at least 32 lie at or above the least of the lanes' largest
// ones (64 at or above the least second largest): there the bisection begins, and it is mostly done after a step or two.
template <int THREADS>
__device__ __forceinline__ unsigned bound_of(const unsigned* __restrict__ keys, int k) {
    const int lane = threadIdx.x & 31;
    unsigned mine[THREADS / 32];
    unsigned first = 0u, second = 0u;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) mine[i] = keys[i * 32 + lane];
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        second = max(second, min(first, mine[i]));
        first = max(first, mine[i]);
    }
    unsigned lo = __reduce_min_sync(0xffffffffu, k <= 32 ? first : second);
    unsigned hi = __reduce_max_sync(0xffffffffu, first);
    const int enough = 2 * k + 8;
    auto above = [&](unsigned bound) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) n += mine[i] >= bound;
        return __reduce_add_sync(0xffffffffu, n);
    };
    if (above(max(lo, KEY_NONE + 1)) <= enough) return lo;
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

// Sum of a count over the block; `sm` is one word of shared memory.
__device__ __forceinline__ int block_count(int n, int* sm) {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (threadIdx.x == 0) *sm = 0;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) atomicAdd(sm, n);
    __syncthreads();
    return *sm;
}

struct __align__(16) Part {              // a chunk's sum of exponentials
    double sum;
    float ref;           // what the exponents were taken against; -infinity: no entry
    int pad;
};

struct ScanArgs {
    const float* logits;
    long long ld;
    int V, k;
    const float* scores;
    Part* part;          // [rows, chunks]
    int2* best;          // [rows, chunks, k]: a logit's bits and its token, descending; -infinity where there are fewer
};

// E logits a thread, held in registers; VEC: four neighbouring ones at a time (rows that start at 16 bytes).  A thread's entries, and
// so the order of a row's sum, depend on their places alone: equal rows have equal sums.
template <int E, bool VEC>
__global__ void __launch_bounds__(ST, 4) beam_scan_kernel(ScanArgs a) {
    ti_pdl_trigger();
    __shared__ double table[16];
    __shared__ unsigned keys[ST];
    __shared__ float warp_top[ST / 32];
    __shared__ double warp_part[ST / 32];
    __shared__ int2 found[ROOM];
    __shared__ int n_found, counter;
    __shared__ unsigned s_bound;
    constexpr int W = VEC ? 4 : 1;           // logits per load
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.y, chunk = blockIdx.x, at = chunk * (ST * E);
    if (tid < 16) table[tid] = __hiloint2double(__double2hiint(pow16[tid]) - (tid << 16), __double2loint(pow16[tid]));
    if (tid == 0) n_found = 0;
    ti_pdl_sync();
    const float* scores = ti_dependent(a.scores);
    const float* x = ti_dependent(a.logits) + (size_t)row * a.ld;
    if (!(scores[row] > -INFINITY)) return;      // (the merge leaves such a row out as well)
    const int end = min(a.V, at + ST * E);
    auto place = [&](int e) { return at + ((e / W) * ST + tid) * W + e % W; };
    float v[E];
    if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const int p = place(e);
            if (p + 4 <= end) {
                const float4 q = *reinterpret_cast<const float4*>(x + p);
                v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[e + j] = p + j < end ? x[p + j] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = place(e) < end ? x[place(e)] : -INFINITY;
    }
    __syncthreads();
    float mine = -INFINITY;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        mine = fmaxf(mine, v[e]);            // (a NaN is passed over)
        s[e & 3] = add_exp(s[e & 3], v[e], table);
    }
    mine = fminf(mine, BIG);
    double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float wtop = warp_max(mine);
    if (lane == 0) {
        warp_top[warp] = wtop;
        warp_part[warp] = sum;
    }
    keys[tid] = order_key(mine);
    __syncthreads();
    float top = warp_top[0];
#pragma unroll
    for (int w = 1; w < ST / 32; ++w) top = fmaxf(top, warp_top[w]);
    const size_t out = (size_t)row * gridDim.x + chunk;
    int2* best = a.best + out * a.k;
    if (top == -INFINITY) {
        if (tid == 0) a.part[out] = Part{0.0, -INFINITY, 0};
        for (int i = tid; i < a.k; i += ST) best[i] = make_int2(__float_as_int(-INFINITY), -1);
        return;
    }
    const bool plain = fabsf(top) <= PLAIN;
    if (!plain) {
        // exponents that would leave the range of 64 bits: once more, against the chunk's largest logit
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (v[e] > -INFINITY) sum += exp((double)fminf(v[e], BIG) - (double)top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) warp_part[warp] = sum;
        __syncthreads();
    }
    if (warp == 0) {
        const unsigned b = bound_of<ST>(keys, a.k);
        if (lane == 0) s_bound = b;
    } else if (tid == 32) {
        double t = warp_part[0];
        for (int w = 1; w < ST / 32; ++w) t += warp_part[w];
        a.part[out] = Part{t, plain ? 0.f : top, 0};
    }
    __syncthreads();
    const unsigned bound = s_bound;
    // f(value, place) for every entry of this thread that counts
    auto each = [&](auto&& f) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (v[e] > -INFINITY) f(fminf(v[e], BIG), place(e));
    };
    auto take = [&](float w, int i) {
        const int to = atomicAdd(&n_found, 1);
        if (to < ROOM) found[to] = make_int2(__float_as_int(w), i);
    };
    if (mine > -INFINITY && order_key(mine) >= bound) each([&](float w, int i) { if (order_key(w) >= bound) take(w, i); });
    __syncthreads();
    int n = n_found;
    if (n > ROOM) {
        // many equal entries: the k-th largest value itself, and of the entries equal to it those with the lowest places
        unsigned lo = bound, hi = order_key(top);
        while (lo < hi) {
            const unsigned mid = lo + ((hi - lo) >> 1) + 1;
            int c = 0;
            each([&](float w, int) { c += order_key(w) >= mid; });
            if (block_count(c, &counter) >= a.k) lo = mid; else hi = mid - 1;
        }
        int c = 0;
        each([&](float w, int) { c += order_key(w) > lo; });
        const int need = a.k - block_count(c, &counter);
        int first = at, last = end - 1;           // the least place up to which `need` entries equal the bound
        while (first < last) {
            const int mid = (first + last) >> 1;
            c = 0;
            each([&](float w, int i) { c += order_key(w) == lo && i <= mid; });
            if (block_count(c, &counter) >= need) last = mid; else first = mid + 1;
        }
        __syncthreads();
        if (tid == 0) n_found = 0;
        __syncthreads();
        each([&](float w, int i) { if (order_key(w) > lo || (order_key(w) == lo && i <= first)) take(w, i); });
        __syncthreads();
        n = min(n_found, ROOM);
    }
    for (int i = tid; i < n; i += ST) {
        const int2 f = found[i];
        const float w = __int_as_float(f.x);
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const int2 g = found[j];
            const float u = __int_as_float(g.x);
            rank += (u > w) | ((u == w) & (g.y < f.y));
        }
        if (rank < a.k) best[rank] = f;
    }
    for (int i = n + tid; i < a.k; i += ST) best[i] = make_int2(__float_as_int(-INFINITY), -1);
}

struct MergeArgs {
    const float* scores;     // [groups, held]
    const Part* part;
    const int2* best;
    const int* stops;
    int held, beams, n_stops, chunks, k, V, ending;
    float* out_score;        // [groups, beams], by place
    int* out_parent;
    int* out_token;
    float* end_score;        // [groups, beams], by rank
    int* end_parent;
    int* end_token;
};

__device__ __forceinline__ unsigned long long order_key64(double x) {
    if (x == 0.0) x = 0.0;
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__global__ void __launch_bounds__(MT) beam_merge_kernel(MergeArgs a) {
    ti_pdl_trigger();
    __shared__ unsigned keys[MT];
    __shared__ unsigned long long found_key[ROOM], found_at[ROOM];   // a total's key; beam << 32 | token, with the top bit for a stop token
    __shared__ double row_ref[BEAMS_MAX], row_log[BEAMS_MAX];        // a row's sum is exp(ref) * exp(log)
    __shared__ float row_score[BEAMS_MAX];
    __shared__ int stops[STOPS_MAX];
    __shared__ float next_score[BEAMS_MAX];
    __shared__ int next_parent[BEAMS_MAX], next_token[BEAMS_MAX], free_place[BEAMS_MAX];
    __shared__ int n_found;
    __shared__ unsigned s_bound;
    __shared__ unsigned long long best_key[MT / 32], best_at[MT / 32];
    constexpr unsigned long long STOP = 1ull << 63;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.x;
    const int lists = a.held * a.chunks, n_all = lists * a.k;
    ti_pdl_sync();
    const float* scores = ti_dependent(a.scores) + (size_t)g * a.held;
    const Part* part = ti_dependent(a.part) + (size_t)g * lists;
    const int2* best = ti_dependent(a.best) + (size_t)g * lists * a.k;
    const int* stop_ids = ti_dependent(a.stops);
    // All entries where they fit the threads' registers, else the first of every list; on their way before anything is waited for.
    const bool whole = n_all <= HELD * MT;
    const int n_items = whole ? n_all : lists, item_step = whole ? 1 : a.k;
    int2 item[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j)
        if (tid + j * MT < n_items) item[j] = best[(size_t)(tid + j * MT) * item_step];
    if (tid < a.n_stops) stops[tid] = stop_ids[tid];
    if (tid < BEAMS_MAX) next_parent[tid] = -1;
    if (tid < a.beams) {
        a.end_score[(size_t)g * a.beams + tid] = -INFINITY;
        a.end_parent[(size_t)g * a.beams + tid] = -1;
        a.end_token[(size_t)g * a.beams + tid] = -1;
    }
    if (tid == 0) n_found = 0;
    for (int b = warp; b < a.held; b += MT / 32) {
        // the logarithm of a row's sum, from its chunks; nearly always all were taken against 0
        const float score = scores[b];
        const Part* p = part + (size_t)b * a.chunks;
        float m = -INFINITY, lowest = INFINITY;
        double t = 0.0;
        for (int c0 = 0; c0 < a.chunks; c0 += 160) {
            Part q[5];
#pragma unroll
            for (int j = 0; j < 5; ++j) q[j] = c0 + j * 32 + lane < a.chunks ? p[c0 + j * 32 + lane] : Part{0.0, -INFINITY, 0};
#pragma unroll
            for (int j = 0; j < 5; ++j) {
                m = fmaxf(m, q[j].ref);
                if (q[j].ref > -INFINITY) {
                    lowest = fminf(lowest, q[j].ref);
                    t += q[j].sum;
                }
            }
        }
        m = warp_max(m);
        lowest = -warp_max(-lowest);
        if (!(score > -INFINITY)) m = -INFINITY;       // (nothing was written for such a row)
        if (m > -INFINITY && lowest < m) {
            t = 0.0;
            for (int c = lane; c < a.chunks; c += 32)
                if (p[c].ref > -INFINITY) t += p[c].sum * exp((double)p[c].ref - (double)m);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) {
            row_score[b] = m > -INFINITY ? score : -INFINITY;
            row_ref[b] = m;
            row_log[b] = m > -INFINITY ? log(t) : 0.0;
        }
    }
    __syncthreads();
    const int per_row = a.chunks * a.k;
    // an entry's total; false where there is none
    auto entry = [&](int beam, int2 f, double& total) {
        const float v = __int_as_float(f.x);
        if (row_score[beam] == -INFINITY || v == -INFINITY) return false;
        total = (double)row_score[beam] + (((double)v - row_ref[beam]) - row_log[beam]);
        return total > -INFINITY;
    };
    auto is_stop = [&](int token) {
        bool stop = false;
        for (int s = 0; s < a.n_stops; ++s) stop |= stops[s] == token;
        return stop;
    };
    auto key_of = [](double t) { return order_key(__double2float_rd(t)); };      // keeps the order, not strictly
    auto take = [&](double total, int beam, int token) {
        const int to = atomicAdd(&n_found, 1);
        if (to < ROOM) {
            found_key[to] = order_key64(total);
            found_at[to] = ((unsigned long long)beam << 32 | (unsigned)token) | (is_stop(token) ? STOP : 0ull);
        }
    };
    const int items_per_row = whole ? per_row : a.chunks;
    unsigned item_key[HELD];
    unsigned mine = KEY_NONE;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        double total;
        const int i = tid + j * MT;
        item_key[j] = 0u;
        if (i < n_items && entry(i / items_per_row, item[j], total)) {
            item_key[j] = key_of(total);
            if (item_key[j] > mine && !is_stop(item[j].y)) mine = item_key[j];
        }
    }
    // (more lists than registers hold: the rest one by one)
    for (int l = tid + HELD * MT; l < n_items; l += MT) {
        double total;
        const int2 f = best[(size_t)l * item_step];
        if (entry(l / items_per_row, f, total) && !is_stop(f.y)) mine = max(mine, key_of(total));
    }
    keys[tid] = mine;
    __syncthreads();
    if (warp == 0) {
        const unsigned b = bound_of<MT>(keys, a.beams);
        if (lane == 0) s_bound = b;
    }
    __syncthreads();
    const unsigned bound = s_bound;
    auto walk = [&](int l, int r) {              // list l from entry r on, down to the bound
        double total;
        for (; r < a.k; ++r) {
            const int2 f = best[(size_t)l * a.k + r];
            if (!entry(l / a.chunks, f, total) || key_of(total) < bound) break;
            take(total, l / a.chunks, f.y);
        }
    };
#pragma unroll
    for (int j = 0; j < HELD; ++j)
        if (item_key[j] >= bound) {              // (an item that is none has key 0, below every bound)
            const int i = tid + j * MT, beam = i / items_per_row;
            double total;
            entry(beam, item[j], total);
            take(total, beam, item[j].y);
            if (!whole) walk(i, 1);
        }
    for (int l = tid + HELD * MT; l < n_items; l += MT) walk(l, 0);
    __syncthreads();
    const int n = n_found;
    const size_t o = (size_t)g * a.beams;
    auto total_of = [](unsigned long long key) {
        return __longlong_as_double((long long)((key >> 63) ? key & 0x7FFFFFFFFFFFFFFFull : ~key));
    };
    auto going = [&](int rank, unsigned long long key, unsigned long long at) {
        next_score[rank] = (float)total_of(key);
        next_parent[rank] = (int)(at >> 32);
        next_token[rank] = (int)at;
    };
    auto ended = [&](int rank, unsigned long long key, unsigned long long at) {
        a.end_score[o + rank] = (float)total_of(key);
        a.end_parent[o + rank] = (int)(at >> 32);
        a.end_token[o + rank] = (int)at;
    };
    if (n <= ROOM) {
        for (int i = tid; i < n; i += MT) {
            const unsigned long long key = found_key[i], whose = found_at[i], at = whose & ~STOP;
            int rank = 0, rank_open = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const unsigned long long k2 = found_key[j], w2 = found_at[j];
                const bool before = (k2 > key) | ((k2 == key) & ((w2 & ~STOP) < at));
                rank += before;
                rank_open += before & (w2 < STOP);
            }
            if (whose < STOP) {
                if (rank_open < a.beams) going(rank_open, key, at);
            } else if (a.ending && rank < a.beams) {
                ended(rank, key, at);
            }
        }
    } else {
        // many equal totals: the candidates one after the other, each the first of those behind the one before
        unsigned long long last_key = ~0ull, last_at = 0;
        for (int rank = 0, open = 0; open < a.beams; ++rank) {
            unsigned long long key = 0, at = ~0ull;          // (the key of a number is never 0)
            for (int i = tid; i < n_all; i += MT) {
                double total;
                const int2 f = best[i];
                if (!entry(i / per_row, f, total)) continue;
                const unsigned long long k2 = order_key64(total), w2 = (unsigned long long)(i / per_row) << 32 | (unsigned)f.y;
                const bool behind = rank == 0 || k2 < last_key || (k2 == last_key && w2 > last_at);
                if (behind && (k2 > key || (k2 == key && w2 < at))) { key = k2; at = w2; }
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, key, d), w2 = __shfl_xor_sync(0xffffffffu, at, d);
                if (k2 > key || (k2 == key && w2 < at)) { key = k2; at = w2; }
            }
            __syncthreads();
            if (lane == 0) { best_key[warp] = key; best_at[warp] = at; }
            __syncthreads();
            for (int w = 0; w < MT / 32; ++w)
                if (best_key[w] > key || (best_key[w] == key && best_at[w] < at)) { key = best_key[w]; at = best_at[w]; }
            if (key == 0) break;                 // no more candidates
            const bool stop = is_stop((int)at);
            if (tid == 0) {
                if (!stop) going(open, key, at);
                else if (a.ending && rank < a.beams) ended(rank, key, at);
            }
            open += !stop;
            last_key = key;
            last_at = at;
        }
    }
    __syncthreads();
    // Placement by one warp, a lane per rank: the first child of a beam stays at its parent's place, the others take the places of
    // the beams without a child, in order.  What is copied is then never what another copy overwrites.
    if (warp == 0) {
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
            a.out_score[o + place] = next_score[lane];
            a.out_parent[o + place] = p;
            a.out_token[o + place] = next_token[lane];
        }
        if (lane < a.beams && !((taken >> lane) & 1u)) {
            a.out_score[o + lane] = -INFINITY;
            a.out_parent[o + lane] = lane;
            a.out_token[o + lane] = 0;
        }
    }
}

// Logits a scan thread holds: the fewest with which the blocks still fit the SMs at once, four each; sixteen at most.
int held_of(int rows, int V) {
    const long long room = 4LL * ti_sm_count();
    for (int e = 4; e < 16; e *= 2)
        if (rows * ((V + ST * e - 1LL) / (ST * e)) <= room) return e;
    return 16;
}

}  // namespace

// Bytes of scratch that ti_beam_select needs.
extern "C" long long ti_beam_select_scratch_bytes(int rows, int V, int beams, int n_stops) {
    if (rows <= 0 || V <= 0 || beams <= 0 || n_stops < 0) return 0;
    const int per = ST * held_of(rows, V), chunks = (V + per - 1) / per;
    const size_t cells = (size_t)rows * chunks;
    return (long long)(cells * sizeof(Part) + cells * (beams + n_stops) * sizeof(int2));
}

// out_scores [2, groups, beams]: the next beams' and the ended ones'; out_places [4, groups, beams]: parents, tokens, and of the
// ended ones parents and tokens.
extern "C" int ti_beam_select(const float* logits, long long ld, int groups, int held, int V, const float* scores, int beams,
                              const int* stops, int n_stops, int ending, float* out_scores, int* out_places, void* scratch,
                              cudaStream_t stream) {
    TI_REQUIRE(groups >= 1 && held >= 1 && V >= 1 && ld >= V, "beam select: %d groups of %d rows of %d logits, %lld apart", groups, held, V, ld);
    TI_REQUIRE(beams >= 1 && beams <= BEAMS_MAX && held <= beams, "beam select: %d beams from %d (at most %d, and no fewer than before)",
               beams, held, BEAMS_MAX);
    TI_REQUIRE(n_stops >= 0 && n_stops <= STOPS_MAX && (n_stops == 0 || stops), "beam select: %d stop tokens (at most %d)", n_stops, STOPS_MAX);
    const long long rows = (long long)groups * held;
    TI_REQUIRE(rows <= 65535, "beam select: %lld rows in one call (at most 65535)", rows);
    TI_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "beam select: the scratch must start at 16 bytes");
    const int e = held_of((int)rows, V), chunks = (V + ST * e - 1) / (ST * e);
    const size_t cells = (size_t)rows * chunks;
    Part* part = static_cast<Part*>(scratch);
    ScanArgs s = {logits, ld, V, beams + n_stops, scores, part, reinterpret_cast<int2*>(part + cells)};
    const bool vec = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    void (*scan)(ScanArgs) = e == 4 ? (vec ? beam_scan_kernel<4, true> : beam_scan_kernel<4, false>)
                           : e == 8 ? (vec ? beam_scan_kernel<8, true> : beam_scan_kernel<8, false>)
                                    : (vec ? beam_scan_kernel<16, true> : beam_scan_kernel<16, false>);
    TI_CUDA(ti_launch(scan, dim3(chunks, (unsigned)rows), dim3(ST), 0, stream, s));
    const size_t n = (size_t)groups * beams;
    MergeArgs m = {scores, s.part, s.best, stops, held, beams, n_stops, chunks, s.k, V, ending,
                   out_scores, out_places, out_places + n, out_scores + n, out_places + 2 * n, out_places + 3 * n};
    TI_CUDA(ti_launch(beam_merge_kernel, dim3(groups), dim3(MT), 0, stream, m));
    return 0;
}
