// Page tables and the map of moves after a beam selection, on the device, from the sequences' lengths and the beams' parents.
//
// A group of beams owns, at every column of the page table that one of them may write, one page per beam ("home").  All beams of a
// group hold the same number of positions L and write the next token into column w = L / PAGE (in a ring of pages: modulo its
// pages).  After a selection a place's sequence is its parent's, so
//
//   * every other column with content takes the parent's page: pages that are not written any more are shared, not copied;
//   * at column w every place needs a page of its own.  A beam that stays keeps the page that it has (of several that share one,
//     as in a ring's older columns, the lowest place keeps it); the others are given, in order, the home pages of the column that
//     nobody keeps, and a move (source page, destination page, rows) of what the column holds already: L mod PAGE rows, or the
//     whole page where the ring has wrapped.
//
// A place whose parent is another place needs that place's state as well: a move (source slot, destination slot, 1).  The selection
// leaves each surviving beam at its place, so no move reads what another one writes; parents that are not so are reported in the
// status word and left out.
//
// A block per group.  Everything here is a few KB: what counts is the launch, so all tables of a cache take one.  A column is read
// and written by one thread, beams first, so the table is changed in place.
#include "tma.cuh"

namespace {
constexpr int BEAMS_MAX = 32;
constexpr int TABLES_MAX = 4;
constexpr int TT = 128;

struct TableArg {
    int* table;              // [slots + 1, width]
    const int* home;         // the same shape: the pages that each slot brought along
    int width, ring_pages;   // ring_pages 0: position p is in column p / PAGE
};

struct TablesArgs {
    TableArg t[TABLES_MAX];
    int n_tables, first;     // first: tables in earlier launches of the same call
    const int* slots;        // [groups, beams]
    const int* parents;
    const int* lengths;      // [groups]
    int extra, groups, beams, page, n_slots;
    int* moves;              // [1 + all tables, groups * beams, 3]
    int* status;
};

__global__ void __launch_bounds__(TT) beam_tables_kernel(TablesArgs a) {
    ti_pdl_trigger();
    __shared__ int slot[BEAMS_MAX], parent[BEAMS_MAX], old_at[BEAMS_MAX];
    const int g = blockIdx.x, tid = threadIdx.x, B = a.beams;
    ti_pdl_sync();
    const int* slots = ti_dependent(a.slots) + (size_t)g * B;
    const int* parents = ti_dependent(a.parents) + (size_t)g * B;
    const int L = ti_dependent(a.lengths)[g] + a.extra;
    if (tid < 32) {
        int p = tid < B ? parents[tid] : tid;
        const int s = tid < B ? slots[tid] : 0;
        const int pp = __shfl_sync(0xffffffffu, p, p & 31);
        const bool bad = tid < B && (p < 0 || p >= B || pp != p || s < 0 || s >= a.n_slots);
        if (bad) {
            ti_report(a.status, TI_STATUS_BEAMS);
            p = tid;
        }
        const bool bad_slot = tid < B && (s < 0 || s >= a.n_slots);
        slot[tid] = bad_slot ? -1 : s;
        parent[tid] = p;
        __syncwarp();
        if (tid < B && slot[parent[tid]] < 0) parent[tid] = tid;
    }
    __syncthreads();
    const size_t at = (size_t)g * B;
    if (a.first == 0 && tid < B) {
        const int p = parent[tid];
        int* m = a.moves + (at + tid) * 3;
        const bool goes = p != tid;
        m[0] = goes ? slot[p] : 0;
        m[1] = goes ? slot[tid] : 0;
        m[2] = goes ? 1 : 0;
    }
    for (int k = 0; k < a.n_tables; ++k) {
        const TableArg t = a.t[k];
        int* table = ti_dependent(t.table);
        const int* home = ti_dependent(t.home);
        const int held = L > 0 ? (L + a.page - 1) / a.page : 0;
        const int used = min(held, t.ring_pages ? min(t.ring_pages, t.width) : t.width);
        const int w = t.ring_pages ? (max(L, 0) / a.page) % t.ring_pages : max(L, 0) / a.page;
        const bool wrapped = t.ring_pages && L >= t.ring_pages * a.page;
        const int rows = wrapped ? a.page : max(L, 0) % a.page;
        const bool begun = w < used;                 // the column that is written next holds something
        for (int c = tid; c < used; c += TT) {
            if (c == w) continue;
            int was[BEAMS_MAX];
#pragma unroll
            for (int b = 0; b < BEAMS_MAX; ++b)
                if (b < B && parent[b] != b) was[b] = table[(size_t)slot[parent[b]] * t.width + c];
#pragma unroll
            for (int b = 0; b < BEAMS_MAX; ++b)
                if (b < B && parent[b] != b) table[(size_t)slot[b] * t.width + c] = was[b];
        }
        if (tid < 32) {
            int* m = a.moves + ((size_t)(1 + a.first + k) * a.groups * B + at + tid) * 3;
            int src = 0, dst = 0, n = 0;
            const bool in = tid < B && begun && slot[tid] >= 0;
            const int p = tid < B ? parent[tid] : tid;
            int page = in ? table[(size_t)slot[p] * t.width + w] : -1 - tid;
            const int mine = in ? home[(size_t)slot[tid] * t.width + w] : -1 - tid;
            // survivors keep their page, the lowest place of those that share one
            const unsigned stays = __ballot_sync(0xffffffffu, in && p == tid);
            const unsigned same = __match_any_sync(0xffffffffu, page);
            const bool keeps = in && p == tid && (__ffs(same & stays) - 1) == tid;
            const unsigned kept = __ballot_sync(0xffffffffu, keeps);
            old_at[tid] = page;
            __syncwarp();
            bool free = in;
            for (int b = 0; b < B; ++b)
                if (((kept >> b) & 1u) && old_at[b] == mine) free = false;
            const unsigned offers = __ballot_sync(0xffffffffu, free);
            const unsigned needs = __ballot_sync(0xffffffffu, in && !keeps);
            const int turn = __popc(needs & ((1u << tid) - 1u));
            const unsigned from = __fns(offers, 0, turn + 1);
            const int given = __shfl_sync(0xffffffffu, mine, from < 32 ? (int)from : tid);
            __syncwarp();
            if (in && !keeps) {
                if (from < 32) {
                    table[(size_t)slot[tid] * t.width + w] = given;
                    if (rows > 0) { src = page; dst = given; n = rows; }
                } else {
                    ti_report(a.status, TI_STATUS_BEAMS);       // the homes do not hold a page per beam
                }
            }
            if (tid < B) { m[0] = src; m[1] = dst; m[2] = n; }
        }
        __syncthreads();
    }
}
}  // namespace

// tables: per table its device address, its home's, its width and its ring's pages, as 64-bit words.
extern "C" int ti_beam_tables(const long long* tables, int n_tables, const int* slots, const int* parents, const int* lengths, int extra,
                              int groups, int beams, int page, int n_slots, int* moves, cudaStream_t stream) {
    TI_REQUIRE(groups >= 1 && beams >= 1 && beams <= BEAMS_MAX, "beam tables: %d groups of %d beams (at most %d)", groups, beams, BEAMS_MAX);
    TI_REQUIRE(n_tables >= 0 && page >= 1 && n_slots >= 1, "beam tables: %d tables of pages of %d", n_tables, page);
    int* status = ti_status_ptr();
    TI_REQUIRE(status != nullptr, "beam tables: no status word");
    for (int first = 0; first == 0 || first < n_tables; first += TABLES_MAX) {
        TablesArgs a = {};
        a.n_tables = n_tables - first < TABLES_MAX ? n_tables - first : TABLES_MAX;
        a.first = first;
        for (int k = 0; k < a.n_tables; ++k) {
            const long long* t = tables + (size_t)(first + k) * 4;
            a.t[k].table = reinterpret_cast<int*>(t[0]);
            a.t[k].home = reinterpret_cast<const int*>(t[1]);
            a.t[k].width = (int)t[2];
            a.t[k].ring_pages = (int)t[3];
        }
        a.slots = slots;
        a.parents = parents;
        a.lengths = lengths;
        a.extra = extra;
        a.groups = groups;
        a.beams = beams;
        a.page = page;
        a.n_slots = n_slots;
        a.moves = moves;
        a.status = status;
        TI_CUDA(ti_launch(beam_tables_kernel, dim3(groups), dim3(TT), 0, stream, a));
    }
    return 0;
}
