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
// leaves each surviving beam at its place, so no move reads what another one writes; parents that are not so, and slots outside the
// tables or twice in a group, are reported in the status word and left out.  A group in which a place goes on from another one, and whose
// homes at column w of any table are not a page of its own for every place, is reported and left as it was, in all tables and states: half
// of a sequence would be another's.  Homes are not written here, so the blocks of a group's tables find the same without waiting for one
// another; and with a page per place there is one for every place that needs one, as the kept pages are homes or leave more of them over.
//
// A block per group and table.  Everything here is a few KB: what counts is the launch and the chain of loads behind it (parents, then
// rows and the pages and homes of column w all at once), so all tables of a cache take one launch, a row is copied by a warp, and its
// first columns are on the way while the homes are looked at: 2.8 us for one request of four beams, 3.3 for 64 of eight over two tables
// of 128 and 16 columns (3.1 and 4.8 with rows and pages read after the homes; 7.4 for the latter with a block per group for all its tables).
#include "tma.cuh"

namespace {
constexpr int BEAMS_MAX = 32;
constexpr int TABLES_MAX = 8;
constexpr int TT = 128;
constexpr int AHEAD = 4;             // columns per lane that are on the way while the homes are looked at

struct TableArg {
    int* table;              // [slots + 1, width]
    const int* home;         // the same shape: the pages that each slot brought along
    int width, ring_pages;   // ring_pages 0: position p is in column p / PAGE
};

struct TablesArgs {
    TableArg t[TABLES_MAX];
    int n_tables;
    const int* slots;        // [groups, beams]
    const int* parents;
    const int* lengths;      // [groups]
    int extra, groups, beams, page, n_slots;
    int* moves;              // [1 + tables, groups * beams, 3]
    int* status;
};

// What a sequence of L positions has in a table: columns in use, the column that its next token goes to, and the rows that it holds there.
struct Column {
    int used, w, rows;
};
__device__ __forceinline__ Column column_of(const TableArg& t, int L, int page) {
    const int pages = L / page;
    Column c;
    c.used = min((L + page - 1) / page, t.ring_pages ? min(t.ring_pages, t.width) : t.width);
    c.w = t.ring_pages ? pages % t.ring_pages : pages;
    c.rows = t.ring_pages && pages >= t.ring_pages ? page : L - pages * page;
    return c;
}

__global__ void __launch_bounds__(TT) beam_tables_kernel(TablesArgs a) {
    ti_pdl_trigger();
    __shared__ int slot[BEAMS_MAX], parent[BEAMS_MAX], moved[BEAMS_MAX], here[BEAMS_MAX];
    __shared__ int s_moved, s_short;
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
        if (lane == 0) {
            s_moved = __popc(goes);
            s_short = 0;
        }
    }
    __syncthreads();
    const int warp = tid >> 5, p = parent[lane], s_own = slot[lane];
    TableArg t = {};
    Column col = {};
    int page = -1 - lane, mine = -1 - lane;      // at column w: what the place's sequence has there, and its home
    int ahead[AHEAD];                            // the first columns of the first row that this warp copies
    if (a.n_tables) {
        t = a.t[blockIdx.y];
        t.table = ti_dependent(t.table);
        col = column_of(t, L, a.page);
        if (warp < s_moved) {
            const int* from = t.table + (size_t)slot[parent[moved[warp]]] * t.width;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) ahead[u] = lane + u * 32 < col.used ? from[lane + u * 32] : 0;
        }
        // a place is short of a page at column w (page 0 is nobody's)
        auto look = [&](const int* home, int width, Column c) {
            const bool in = lane < B && c.w < c.used && s_own >= 0;
            const int of = in ? ti_dependent(home)[(size_t)s_own * width + c.w] : -1 - lane;
            const unsigned twins = __match_any_sync(0xffffffffu, of);
            if (in && s_moved && (of <= 0 || (twins & (twins - 1u)))) s_short = 1;
            return of;
        };
        if (warp == 0) {
            if (lane < B && col.w < col.used && s_own >= 0) page = t.table[(size_t)slot[p] * t.width + col.w];
            mine = look(t.home, t.width, col);
        }
        for (int k = warp ? warp : TT / 32; k < a.n_tables; k += TT / 32) {
            const TableArg& other = a.t[blockIdx.y + k < a.n_tables ? blockIdx.y + k : blockIdx.y + k - a.n_tables];
            look(other.home, other.width, column_of(other, L, a.page));
        }
    }
    __syncthreads();
    const bool left = s_short != 0;
    if (left && tid == 0) ti_report(a.status, TI_STATUS_BEAMS);
    if (blockIdx.y == 0 && tid < B) {
        const bool goes = p != lane && !left;
        int* m = a.moves + (at + lane) * 3;
        m[0] = goes ? slot[p] : 0;
        m[1] = goes ? s_own : 0;
        m[2] = goes ? 1 : 0;
    }
    if (a.n_tables == 0) return;
    int* m = a.moves + ((size_t)(1 + blockIdx.y) * a.groups * B + at + lane) * 3;
    if (left) {
        if (tid < B) m[0] = m[1] = m[2] = 0;
        return;
    }
    const int used = col.used, w = col.w, rows = col.rows;
    // A survivor's row stays as it is at every column but w, and only survivors' rows are read: no order matters.
    for (int j = warp; j < s_moved; j += TT / 32) {
        const int* from = t.table + (size_t)slot[parent[moved[j]]] * t.width;
        int* to = t.table + (size_t)slot[moved[j]] * t.width;
        int c = lane;
        if (j == warp)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u, c += 32)
                if (c < used && c != w) to[c] = ahead[u];
#pragma unroll 4
        for (; c < used; c += 32)
            if (c != w) to[c] = from[c];
    }
    if (warp != 0) return;
    const bool in = lane < B && w < used && s_own >= 0;              // the column that is written next holds something
    const unsigned below = (1u << lane) - 1u;
    // survivors keep their page, the lowest place of those that share one
    const unsigned stays = __ballot_sync(0xffffffffu, in && p == lane);
    const unsigned same = __match_any_sync(0xffffffffu, page);
    const bool keeps = in && p == lane && !(same & stays & below);
    const unsigned kept = __ballot_sync(0xffffffffu, keeps);
    const unsigned like_mine = __match_any_sync(0xffffffffu, mine);
    bool free = in && mine > 0 && !(like_mine & below);
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
            t.table[(size_t)s_own * t.width + w] = given;
            if (rows > 0) { src = page; dst = given; n = rows; }
        } else {
            ti_report(a.status, TI_STATUS_BEAMS);                    // (nobody moves, two share a page, and there is none for one of them)
        }
    }
    if (lane < B) { m[0] = src; m[1] = dst; m[2] = n; }
}
}  // namespace

// tables: per table its device address, its home's, its width and its ring's pages, as 64-bit words.
extern "C" int ti_beam_tables(const long long* tables, int n_tables, const int* slots, const int* parents, const int* lengths, int extra,
                              int groups, int beams, int page, int n_slots, int* moves, cudaStream_t stream) {
    TI_REQUIRE(groups >= 1 && beams >= 1 && beams <= BEAMS_MAX, "beam tables: %d groups of %d beams (at most %d)", groups, beams, BEAMS_MAX);
    TI_REQUIRE(n_tables >= 0 && n_tables <= TABLES_MAX && page >= 1 && n_slots >= 1, "beam tables: %d tables (at most %d) of pages of %d", n_tables,
               TABLES_MAX, page);
    int* status = ti_status_ptr();
    TI_REQUIRE(status != nullptr, "beam tables: no status word");
    TablesArgs a = {};
    a.n_tables = n_tables;
    for (int k = 0; k < n_tables; ++k) {
        const long long* t = tables + (size_t)k * 4;
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
    TI_CUDA(ti_launch(beam_tables_kernel, dim3(groups, n_tables ? n_tables : 1), dim3(TT), 0, stream, a));
    return 0;
}
