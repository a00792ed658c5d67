// Beam search's selection: from the logits of every beam and the beams' scores to the next beams.
//
//   total(g, b, v) = score(g, b) + (x(b, v) - m(b)) - log sum_u exp(x(b, u) - m(b)),   m(b) the largest logit of the row
//
// A group's candidates are ordered by total, descending, and by (b, v) where totals are equal.  The first ``beams`` of them whose
// token is no stop token go on; those among the first ``beams`` of all whose token is one have ended.  NaN counts as -infinity,
// +infinity as the largest finite number; a candidate at -infinity is none, so masked tokens and beams at -infinity never win.
//
// Two kernels.  The scan runs blocks over (chunk, row): a chunk's logits are read once, into registers; from there come its largest
// value, its sum of exponentials against that, and its best K = beams + stop tokens entries (at most that many of one row can
// matter: of the first ``beams`` entries that are no stop tokens all but the stop tokens before them).  The merge runs a block per
// group over what the scan left.
//
// The best K of a chunk without sorting it: the K-th largest of the threads' own maxima is a lower bound of the K-th largest
// entry, and few entries lie above it; those are gathered and ranked by counting.  The merge finds its ``beams`` in the same way.
// Where so many entries are equal that the gathered ones overflow their room, the bound is made exact entry by entry.
//
// Totals, sums and the order are in 64 bits: beams compete by sums over a whole vocabulary, and at 32 bits the order of two
// candidates of different rows would depend on how the sums were split.
#include "common.cuh"

#include <climits>

namespace {
constexpr int BEAMS_MAX = 32;        // a group's beams: one bit of a warp's word each
constexpr int STOPS_MAX = 16;
constexpr int ST = 256;              // threads of a scan block
constexpr int ROOM = 1024;           // entries above the bound that a block can rank
constexpr int MT = 512;              // threads of a merge block

__device__ __forceinline__ unsigned order_key(float x) {
    if (x == 0.f) x = 0.f;      // -0 counts as +0
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr unsigned KEY_NONE = 0x007FFFFFu;      // the key of -infinity: the least key of all

// A value at or below the k-th largest of the block's keys (one per thread, in shared memory), with few keys more above it than k:
// bisection between the least and the largest key, the same in every warp.
template <int THREADS>
__device__ __forceinline__ unsigned bound_of(const unsigned* __restrict__ keys, int k) {
    const int lane = threadIdx.x & 31;
    unsigned mine[THREADS / 32];
    unsigned lo = ~0u, hi = 0u;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        mine[i] = keys[i * 32 + lane];
        lo = min(lo, mine[i]);
        hi = max(hi, mine[i]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    const int enough = k + (k >> 1) + 2;
    while (lo < hi) {
        const unsigned mid = lo + ((hi - lo) >> 1) + 1;
        int n = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) n += mine[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
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

struct ScanArgs {
    const float* logits;
    long long ld;
    int V, chunk, k;
    const float* scores;
    float* top;          // [rows, chunks]
    double* sum;         // [rows, chunks]
    int2* best;          // [rows, chunks, k]: a logit's bits and its token, descending; -infinity where there are fewer
};

// E logits per thread; VEC: four neighbouring ones at a time (rows that start at 16 bytes).
template <int E, bool VEC>
__global__ void __launch_bounds__(ST) beam_scan_kernel(ScanArgs a) {
    ti_pdl_trigger();
    __shared__ unsigned keys[ST];
    __shared__ float warp_top[ST / 32];
    __shared__ double warp_sum_[ST / 32];
    __shared__ int2 found[ROOM];
    __shared__ int n_found, counter;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.y, chunk = blockIdx.x, at = chunk * a.chunk;
    ti_pdl_sync();
    const float* scores = ti_dependent(a.scores);
    const float* x = ti_dependent(a.logits) + (size_t)row * a.ld;
    if (!(scores[row] > -INFINITY)) return;      // (the merge leaves such a row out as well)
    const int end = min(a.V, at + a.chunk);
    auto place = [&](int e) { return VEC ? at + ((e >> 2) * ST + tid) * 4 + (e & 3) : at + e * ST + tid; };
    float v[E];
    if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const int i = place(e);
            if (i + 4 <= end) {
                const float4 q = *reinterpret_cast<const float4*>(x + i);
                v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[e + j] = i + j < end ? x[i + j] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = place(e);
            v[e] = i < end ? x[i] : -INFINITY;
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = v[e] >= -INFINITY ? fminf(v[e], 3.402823466e38f) : -INFINITY;       // (NaN compares false)
        mine = fmaxf(mine, v[e]);
    }
    const float wtop = warp_max(mine);
    if (lane == 0) warp_top[warp] = wtop;
    keys[tid] = order_key(mine);
    if (tid == 0) n_found = 0;
    __syncthreads();
    float top = warp_top[0];
#pragma unroll
    for (int w = 1; w < ST / 32; ++w) top = fmaxf(top, warp_top[w]);
    const size_t out = (size_t)row * gridDim.x + chunk;
    int2* best = a.best + out * a.k;
    if (top == -INFINITY) {
        if (tid == 0) a.top[out] = -INFINITY;
        if (tid == 0) a.sum[out] = 0.0;
        for (int i = tid; i < a.k; i += ST) best[i] = make_int2(__float_as_int(-INFINITY), -1);
        return;
    }

    double sum = 0.0;
#pragma unroll 4
    for (int e = 0; e < E; ++e) sum += exp((double)v[e] - (double)top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum_[warp] = sum;

    unsigned bound = bound_of<ST>(keys, a.k);
    auto gather = [&](auto&& wanted) {
        int n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += wanted(v[e], place(e));
        if (n) {
            int to = atomicAdd(&n_found, n);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (wanted(v[e], place(e))) {
                    if (to < ROOM) found[to] = make_int2(__float_as_int(v[e]), place(e));
                    ++to;
                }
        }
    };
    if (order_key(mine) >= bound) gather([&](float w, int) { return w > -INFINITY && order_key(w) >= bound; });
    __syncthreads();
    int n = n_found;
    if (n > ROOM) {
        // many equal entries: the k-th largest value itself, and of the entries equal to it those with the lowest places
        unsigned lo = bound, hi = order_key(top);
        while (lo < hi) {
            const unsigned mid = lo + ((hi - lo) >> 1) + 1;
            int c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c += v[e] > -INFINITY && order_key(v[e]) >= mid;
            if (block_count(c, &counter) >= a.k) lo = mid; else hi = mid - 1;
        }
        int c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) c += order_key(v[e]) > lo;
        const int need = a.k - block_count(c, &counter);
        int first = at, last = end - 1;           // the least place up to which `need` entries equal the bound
        while (first < last) {
            const int mid = (first + last) >> 1;
            c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c += order_key(v[e]) == lo && place(e) <= mid;
            if (block_count(c, &counter) >= need) last = mid; else first = mid + 1;
        }
        __syncthreads();
        if (tid == 0) n_found = 0;
        __syncthreads();
        gather([&](float w, int i) { return order_key(w) > lo || (order_key(w) == lo && i <= first && w > -INFINITY); });
        __syncthreads();
        n = min(n_found, ROOM);
    }
    for (int i = tid; i < n; i += ST) {
        const int2 f = found[i];
        const float w = __int_as_float(f.x);
        int rank = 0;
        for (int j = 0; j < n; ++j) {
            const int2 g = found[j];
            const float u = __int_as_float(g.x);
            rank += u > w || (u == w && g.y < f.y);
        }
        if (rank < a.k) best[rank] = f;
    }
    for (int i = n + tid; i < a.k; i += ST) best[i] = make_int2(__float_as_int(-INFINITY), -1);
    if (tid == 0) {
        double s = warp_sum_[0];
        for (int w = 1; w < ST / 32; ++w) s += warp_sum_[w];
        a.top[out] = top;
        a.sum[out] = s;
    }
}

struct MergeArgs {
    const float* scores;     // [groups, held]
    const float* top;
    const double* sum;
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

struct Candidate {
    double total;
    int beam, token;         // token -1 - t for a stop token t
};

__device__ __forceinline__ bool before(double t, int beam, int token, double t2, int beam2, int token2) {
    return t > t2 || (t == t2 && (beam < beam2 || (beam == beam2 && token < token2)));
}

__global__ void __launch_bounds__(MT) beam_merge_kernel(MergeArgs a) {
    ti_pdl_trigger();
    __shared__ unsigned keys[MT];
    __shared__ Candidate found[ROOM];
    __shared__ double row_add[BEAMS_MAX];         // score - log of the row's sum
    __shared__ float row_top[BEAMS_MAX];
    __shared__ int stops[STOPS_MAX];
    __shared__ double next_total[BEAMS_MAX];
    __shared__ int next_parent[BEAMS_MAX], next_token[BEAMS_MAX];
    __shared__ int n_found;
    __shared__ double best_total[MT / 32];
    __shared__ int best_beam[MT / 32], best_token[MT / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.x;
    ti_pdl_sync();
    const float* scores = ti_dependent(a.scores) + (size_t)g * a.held;
    const float* top = ti_dependent(a.top) + (size_t)g * a.held * a.chunks;
    const double* sum = ti_dependent(a.sum) + (size_t)g * a.held * a.chunks;
    const int2* best = ti_dependent(a.best) + (size_t)g * a.held * a.chunks * a.k;
    const int* stop_ids = ti_dependent(a.stops);
    if (tid < a.n_stops) stops[tid] = stop_ids[tid];
    if (tid < BEAMS_MAX) {
        next_total[tid] = -INFINITY;
        next_parent[tid] = -1;
    }
    if (tid < a.beams) {
        a.end_score[(size_t)g * a.beams + tid] = -INFINITY;
        a.end_parent[(size_t)g * a.beams + tid] = -1;
        a.end_token[(size_t)g * a.beams + tid] = -1;
    }
    if (tid == 0) n_found = 0;
    for (int b = warp; b < a.held; b += MT / 32) {
        // a row's largest logit and the logarithm of its sum, from its chunks
        const float score = scores[b];
        if (!(score > -INFINITY)) {
            if (lane == 0) { row_top[b] = -INFINITY; row_add[b] = -INFINITY; }
            continue;
        }
        float m = -INFINITY;
        for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, top[b * a.chunks + c]);
        m = warp_max(m);
        double s = 0.0;
        if (m > -INFINITY)
            for (int c = lane; c < a.chunks; c += 32) s += sum[b * a.chunks + c] * exp((double)top[b * a.chunks + c] - (double)m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) { row_top[b] = m; row_add[b] = m > -INFINITY ? -log(s) : -INFINITY; }
    }
    __syncthreads();
    const int per_row = a.chunks * a.k, n_all = a.held * per_row;
    // candidate i: its beam, token (negative for a stop token) and total; false where there is none
    auto candidate = [&](int i, Candidate& c) {
        c.beam = i / per_row;
        const float m = row_top[c.beam];
        if (m == -INFINITY) return false;
        const int2 f = best[i];
        const float v = __int_as_float(f.x);
        if (v == -INFINITY) return false;
        c.total = (double)scores[c.beam] + (((double)v - (double)m) + row_add[c.beam]);
        c.token = f.y;
        for (int s = 0; s < a.n_stops; ++s)
            if (stops[s] == f.y) c.token = -1 - f.y;
        return c.total > -INFINITY;
    };
    auto key_of = [](double t) { return order_key(__double2float_rd(t)); };      // keeps the order, not strictly
    unsigned mine = KEY_NONE;
    for (int i = tid; i < n_all; i += MT) {
        Candidate c;
        if (candidate(i, c) && c.token >= 0) mine = max(mine, key_of(c.total));
    }
    keys[tid] = mine;
    __syncthreads();
    const unsigned bound = bound_of<MT>(keys, a.beams);
    for (int i = tid; i < n_all; i += MT) {
        Candidate c;
        if (candidate(i, c) && key_of(c.total) >= bound) {
            const int to = atomicAdd(&n_found, 1);
            if (to < ROOM) found[to] = c;
        }
    }
    __syncthreads();
    int n = n_found;
    if (n <= ROOM) {
        for (int i = tid; i < n; i += MT) {
            const Candidate c = found[i];
            const int token = c.token < 0 ? -1 - c.token : c.token;
            int rank = 0, rank_open = 0;
            for (int j = 0; j < n; ++j) {
                const Candidate d = found[j];
                const bool b = before(d.total, d.beam, d.token < 0 ? -1 - d.token : d.token, c.total, c.beam, token);
                rank += b;
                rank_open += b && d.token >= 0;
            }
            if (c.token >= 0 && rank_open < a.beams) {
                next_total[rank_open] = c.total;
                next_parent[rank_open] = c.beam;
                next_token[rank_open] = token;
            } else if (c.token < 0 && a.ending && rank < a.beams) {
                a.end_score[(size_t)g * a.beams + rank] = (float)c.total;
                a.end_parent[(size_t)g * a.beams + rank] = c.beam;
                a.end_token[(size_t)g * a.beams + rank] = token;
            }
        }
    } else {
        // many equal totals: the candidates one after the other, each the first of those behind the one before
        double last = INFINITY;
        int last_beam = -1, last_token = -1, open = 0;
        for (int rank = 0; open < a.beams; ++rank) {
            double t = -INFINITY;
            int beam = INT_MAX, token = INT_MAX;
            for (int i = tid; i < n_all; i += MT) {
                Candidate c;
                if (!candidate(i, c)) continue;
                const int tok = c.token < 0 ? -1 - c.token : c.token;
                if ((rank == 0 || before(last, last_beam, last_token, c.total, c.beam, tok)) && before(c.total, c.beam, tok, t, beam, token)) {
                    t = c.total; beam = c.beam; token = tok;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const double t2 = __shfl_xor_sync(0xffffffffu, t, o);
                const int b2 = __shfl_xor_sync(0xffffffffu, beam, o), k2 = __shfl_xor_sync(0xffffffffu, token, o);
                if (before(t2, b2, k2, t, beam, token)) { t = t2; beam = b2; token = k2; }
            }
            __syncthreads();
            if (lane == 0) { best_total[warp] = t; best_beam[warp] = beam; best_token[warp] = token; }
            __syncthreads();
            t = best_total[0]; beam = best_beam[0]; token = best_token[0];
            for (int w = 1; w < MT / 32; ++w)
                if (before(best_total[w], best_beam[w], best_token[w], t, beam, token)) { t = best_total[w]; beam = best_beam[w]; token = best_token[w]; }
            if (beam == INT_MAX) break;          // no more candidates
            bool stop = false;
            for (int s = 0; s < a.n_stops; ++s) stop |= stops[s] == token;
            if (tid == 0) {
                if (!stop) {
                    next_total[open] = t; next_parent[open] = beam; next_token[open] = token;
                } else if (a.ending && rank < a.beams) {
                    a.end_score[(size_t)g * a.beams + rank] = (float)t;
                    a.end_parent[(size_t)g * a.beams + rank] = beam;
                    a.end_token[(size_t)g * a.beams + rank] = token;
                }
            }
            open += !stop;
            last = t; last_beam = beam; last_token = token;
        }
    }
    __syncthreads();
    // Placement by one warp, a lane per rank: the first child of a beam stays at its parent's place, the others take the places of
    // the beams without a child, in order.  What is copied is then never what another copy overwrites.
    if (warp == 0) {
        const int p = next_parent[lane];
        const bool there = p >= 0;
        const unsigned same = __match_any_sync(0xffffffffu, p);
        const bool stays = there && (__ffs(same) - 1) == lane;
        const unsigned kept = __reduce_or_sync(0xffffffffu, stays ? 1u << p : 0u);
        const unsigned goes = __ballot_sync(0xffffffffu, there && !stays);
        const unsigned here = __ballot_sync(0xffffffffu, stays);
        int place = -1;
        if (stays) place = p;
        else if (there) place = __fns(~kept, 0, __popc(goes & ((1u << lane) - 1u)) + 1);
        const unsigned taken = __reduce_or_sync(0xffffffffu, place >= 0 ? 1u << place : 0u);
        (void)here;
        const size_t o = (size_t)g * a.beams;
        if (place >= 0) {
            a.out_score[o + place] = (float)next_total[lane];
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

// Logits per scan block.
int chunk_of(int rows, int V) {
    (void)rows; (void)V;
    return ST * 32;
}

size_t align16(size_t n) { return (n + 15) & ~size_t(15); }
}  // namespace

// Bytes of scratch that ti_beam_select needs.
extern "C" long long ti_beam_select_scratch_bytes(int rows, int V, int beams, int n_stops) {
    if (rows <= 0 || V <= 0 || beams <= 0 || n_stops < 0) return 0;
    const int per = chunk_of(rows, V), chunks = (V + per - 1) / per;
    const size_t cells = (size_t)rows * chunks;
    return (long long)(align16(cells * 4) + align16(cells * 8) + cells * (beams + n_stops) * 8);
}

extern "C" int ti_beam_select(const float* logits, long long ld, int groups, int held, int V, const float* scores, int beams,
                              const int* stops, int n_stops, int ending, float* out_score, int* out_parent, int* out_token,
                              float* end_score, int* end_parent, int* end_token, void* scratch, cudaStream_t stream) {
    TI_REQUIRE(groups >= 1 && held >= 1 && V >= 1 && ld >= V, "beam select: %d groups of %d rows of %d logits, %lld apart", groups, held, V, ld);
    TI_REQUIRE(beams >= 1 && beams <= BEAMS_MAX && held <= beams, "beam select: %d beams from %d (at most %d, and no fewer than before)",
               beams, held, BEAMS_MAX);
    TI_REQUIRE(n_stops >= 0 && n_stops <= STOPS_MAX && (n_stops == 0 || stops), "beam select: %d stop tokens (at most %d)", n_stops, STOPS_MAX);
    const long long rows = (long long)groups * held;
    TI_REQUIRE(rows <= 65535, "beam select: %lld rows in one call (at most 65535)", rows);
    TI_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "beam select: the scratch must start at 16 bytes");
    const int per = chunk_of((int)rows, V), chunks = (V + per - 1) / per;
    const size_t cells = (size_t)rows * chunks;
    char* at = static_cast<char*>(scratch);
    ScanArgs s = {logits, ld, V, per, beams + n_stops, scores, nullptr, nullptr, nullptr};
    s.top = reinterpret_cast<float*>(at);
    s.sum = reinterpret_cast<double*>(at + align16(cells * 4));
    s.best = reinterpret_cast<int2*>(at + align16(cells * 4) + align16(cells * 8));
    const bool vec = ld % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    const dim3 grid(chunks, (unsigned)rows);
    TI_CUDA(ti_launch(vec ? beam_scan_kernel<32, true> : beam_scan_kernel<32, false>, grid, dim3(ST), 0, stream, s));
    MergeArgs m = {scores, s.top, s.sum, s.best, stops, held, beams, n_stops, chunks, s.k, V, ending,
                   out_score, out_parent, out_token, end_score, end_parent, end_token};
    TI_CUDA(ti_launch(beam_merge_kernel, dim3(groups), dim3(MT), 0, stream, m));
    return 0;
}
