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
// leaves each surviving beam at its place, so no move reads what another one writes; parents that are not so, slots outside the
// tables or twice in a group, and homes without a page per beam are reported in the status word and left out.
//
// A block per group and table.  Everything here is a few KB: what counts is the launch and the chain of loads behind it (parents,
// then rows, then the pages of column w), so all tables of a cache take one launch and a row is copied by a warp: 2.4 us for one request
// of four beams, 4.0 for 64 of eight over two tables of 128 and 16 columns (4.2 and 7.4 with a block per group for all its tables).
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
    __shared__ int slot[BEAMS_MAX], parent[BEAMS_MAX], moved[BEAMS_MAX], here[BEAMS_MAX];
    __shared__ int s_moved;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, B = a.beams;
    const size_t at = (size_t)g * B;
    ti_pdl_sync();
    const int L = max(ti_dependent(a.lengths)[g] + a.extra, 0);
    if (tid < 32) {
        int p = lane < B ? ti_dependent(a.parents)[at + lane] : lane;
        const int s = lane < B ? ti_dependent(a.slots)[at + lane] : 0;
        const unsigned twins = __match_any_sync(0xffffffffu, lane < B ? s : -1 - lane);
        const bool slot_ok = s >= 0 && s < a.n_slots && (twins & (twins - 1u)) == 0u;        // a slot of its own
        const int pp = __shfl_sync(0xffffffffu, p, p & 31);
        const bool source_ok = __shfl_sync(0xffffffffu, (int)slot_ok, p & 31);
        if (lane < B && (p < 0 || p >= B || pp != p || !slot_ok || !source_ok)) {
            ti_report(a.status, TI_STATUS_BEAMS);
            p = lane;
        }
        slot[lane] = slot_ok ? s : -1;
        parent[lane] = p;
        const unsigned goes = __ballot_sync(0xffffffffu, p != lane);
        if (p != lane) moved[__popc(goes & ((1u << lane) - 1u))] = lane;
        if (lane == 0) s_moved = __popc(goes);
        __syncwarp();
        if (blockIdx.y == 0 && a.first == 0 && lane < B) {
            int* m = a.moves + (at + lane) * 3;
            m[0] = p != lane ? slot[p] : 0;
            m[1] = p != lane ? s : 0;
            m[2] = p != lane ? 1 : 0;
        }
    }
    if (a.n_tables == 0) return;
    __syncthreads();
    const TableArg t = a.t[blockIdx.y];
    int* table = ti_dependent(t.table);
    const int pages = L / a.page;
    const int used = min((L + a.page - 1) / a.page, t.ring_pages ? min(t.ring_pages, t.width) : t.width);
    const int w = t.ring_pages ? pages % t.ring_pages : pages;
    const int rows = t.ring_pages && pages >= t.ring_pages ? a.page : L - pages * a.page;
    // A survivor's row stays as it is at every column but w, and only survivors' rows are read: no order matters.
    for (int j = tid >> 5; j < s_moved; j += TT / 32) {
        const int* from = table + (size_t)slot[parent[moved[j]]] * t.width;
        int* to = table + (size_t)slot[moved[j]] * t.width;
#pragma unroll 4
        for (int c = lane; c < used; c += 32)
            if (c != w) to[c] = from[c];
    }
    if (tid >= 32) return;
    int* m = a.moves + ((size_t)(1 + a.first + blockIdx.y) * a.groups * B + at + lane) * 3;
    const bool in = lane < B && w < used && slot[lane] >= 0;         // the column that is written next holds something
    const int p = parent[lane];
    const int page = in ? table[(size_t)slot[p] * t.width + w] : -1 - lane;
    const int mine = in ? ti_dependent(t.home)[(size_t)slot[lane] * t.width + w] : -1 - lane;
    const unsigned below = (1u << lane) - 1u;
    // survivors keep their page, the lowest place of those that share one
    const unsigned stays = __ballot_sync(0xffffffffu, in && p == lane);
    const unsigned same = __match_any_sync(0xffffffffu, page);
    const bool keeps = in && p == lane && !(same & stays & below);
    const unsigned kept = __ballot_sync(0xffffffffu, keeps);
    bool free = in && mine > 0;                                      // (page 0 is nobody's)
    for (unsigned k = kept; k; k &= k - 1u)
        if (__shfl_sync(0xffffffffu, page, __ffs(k) - 1) == mine) free = false;
    const unsigned offers = __ballot_sync(0xffffffffu, free), needs = __ballot_sync(0xffffffffu, in && !keeps);
    if (free) here[__popc(offers & below)] = mine;
    __syncwarp();                                                    // (every page has been read: rows may change)
    int src = 0, dst = 0, n = 0;
    if (in && !keeps) {
        const int turn = __popc(needs & below);
        if (turn < __popc(offers)) {
            const int given = here[turn];
            table[(size_t)slot[lane] * t.width + w] = given;
            if (rows > 0) { src = page; dst = given; n = rows; }
        } else {
            ti_report(a.status, TI_STATUS_BEAMS);                    // the homes do not hold a page per beam
        }
    }
    if (lane < B) { m[0] = src; m[1] = dst; m[2] = n; }
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
        TI_CUDA(ti_launch(beam_tables_kernel, dim3(groups, a.n_tables ? a.n_tables : 1), dim3(TT), 0, stream, a));
    }
    return 0;
}
