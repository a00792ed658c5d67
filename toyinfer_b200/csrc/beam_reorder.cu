// Moves what beams take over from their parents: rows of the pages that are being written, and whole states, of all layers at once.
//
// An area is a tensor of equal units (pages of a group of layers, slots of a state): unit u of a run starts at
// base + outer * o + inner * i + u * unit, and its first n rows of `row` bytes follow one another.  A move (source unit, destination
// unit, n) of an area's list copies those rows of every run.  The moves are on the device (beam_tables.cu); the host knows neither
// how many there are nor how long they are.
//
// A unit outside the tensor is reported in the status word, and nothing is moved for it.
//
// The only work is bytes: each is read once and written once.  Warps take pieces of PIECE bytes, all pieces of all runs of all moves
// in one numbering, so a few moves of a small cache spread over the SMs as many moves of a large one do.  Widths of 16, 4 or 2
// bytes, as the area's addresses and strides allow; a warp has eight loads on the way before its first store.  Four blocks an SM, all
// resident, and pieces as long as a head's page keep what DRAM reads and writes in long runs: 32 moves of part pages of 36 layers (261
// MB read and written) take 43.5 us; 46.1 with pieces of 8 KB, 45.8 with five blocks, 48.5 with three, 73 with sixteen loads on the
// way; 39.9 at the copy rate.  Twelve states of 38 MB that start at any 4 bytes (911 MB) take 151.7 us, 139 at the copy rate.
#include "tma.cuh"

namespace {
constexpr int LISTS_MAX = 9;         // states, and up to eight page tables
constexpr int RT = 256;
constexpr int PIECE = 16384;         // a page of 64 rows of 128 elements of 16 bits
constexpr int BLOCKS = 4;            // an SM, all at once

struct Area {                        // as the host writes it: 64-bit words
    long long base, outer, n_outer, inner, n_inner, unit, units, row, rows, width, pieces, first;
};  // units: how many; rows: of a whole unit; width: bytes per access; pieces: of one run; first: pieces of its list's areas before it

struct ReorderArgs {
    const Area* areas;
    int n_areas, n_lists, n_moves;
    const int* moves;                // [lists, n_moves, 3]
    int first_area[LISTS_MAX + 1];   // areas are sorted by list
    long long pieces[LISTS_MAX];     // pieces of one move, over the areas of the list
    int* status;
};

template <typename V>
__device__ __forceinline__ void copy_piece(char* dst, const char* src, int bytes, int lane) {
    const int n = bytes / (int)sizeof(V);
    const V* s = reinterpret_cast<const V*>(src);
    V* d = reinterpret_cast<V*>(dst);
    int i = lane;
    for (; i + 7 * 32 < n; i += 8 * 32) {
        V v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s[i + j * 32];
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i + j * 32] = v[j];
    }
    for (; i < n; i += 32) d[i] = s[i];
}

// It lets no later kernel start before it ends: attention kernels read page tables and earlier rows before they wait for the kernel
// before them, as no other kernel writes those.
__global__ void __launch_bounds__(RT) beam_reorder_kernel(ReorderArgs a) {
    extern __shared__ int active[];          // [lists, n_moves]: the moves that copy something
    __shared__ int count[LISTS_MAX];
    ti_pdl_sync();
    const int* moves = ti_dependent(a.moves);
    const Area* areas = ti_dependent(a.areas);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int l = warp; l < a.n_lists; l += RT / 32) {
        int n = 0;
        for (int i = lane; i - lane < a.n_moves; i += 32) {
            const bool on = i < a.n_moves && moves[((size_t)l * a.n_moves + i) * 3 + 2] > 0;
            const unsigned b = __ballot_sync(0xffffffffu, on);
            if (on) active[l * a.n_moves + n + __popc(b & ((1u << lane) - 1u))] = i;
            n += __popc(b);
        }
        if (lane == 0) count[l] = n;
    }
    __syncthreads();
    long long total = 0;
    for (int l = 0; l < a.n_lists; ++l) total += count[l] * a.pieces[l];
    const long long step = (long long)gridDim.x * (RT / 32);
    for (long long at = (long long)blockIdx.x * (RT / 32) + warp; at < total; at += step) {
        long long r = at;
        int l = 0;
        for (; r >= count[l] * a.pieces[l]; ++l) r -= count[l] * a.pieces[l];
        const int m = active[l * a.n_moves + (int)(r / a.pieces[l])];
        r %= a.pieces[l];
        int lo = a.first_area[l], hi = a.first_area[l + 1] - 1;
        while (lo < hi) {                    // the last area that begins at or before r
            const int mid = (lo + hi + 1) >> 1;
            if (areas[mid].first <= r) lo = mid; else hi = mid - 1;
        }
        const Area* A = areas + lo;
        r -= A->first;
        const int* mv = moves + ((size_t)l * a.n_moves + m) * 3;
        const int src = mv[0], dst = mv[1], rows = (int)min((long long)mv[2], A->rows);
        if (src < 0 || dst < 0 || src >= A->units || dst >= A->units) {
            if (lane == 0) ti_report(a.status, TI_STATUS_BEAMS);
            continue;
        }
        const int piece = (int)(r % A->pieces);
        const long long run = r / A->pieces;
        const long long all = rows * A->row, from = (long long)piece * PIECE;
        if (from >= all) continue;
        const int bytes = (int)min((long long)PIECE, all - from);
        char* base = reinterpret_cast<char*>(A->base) + (run / A->n_inner) * A->outer + (run % A->n_inner) * A->inner + from;
        const char* s = base + src * A->unit;
        char* d = base + dst * A->unit;
        if (A->width == 16) copy_piece<int4>(d, s, bytes, lane);
        else if (A->width == 4) copy_piece<int>(d, s, bytes, lane);
        else copy_piece<short>(d, s, bytes, lane);
    }
}
}  // namespace

// areas: device address of n_areas records; first_area [lists + 1] and pieces [lists] on the host.
extern "C" int ti_beam_reorder(const void* areas, int n_areas, int n_lists, const int* first_area, const long long* pieces, const int* moves,
                               int n_moves, cudaStream_t stream) {
    TI_REQUIRE(n_lists >= 1 && n_lists <= LISTS_MAX, "beam reorder: %d lists of moves (at most %d)", n_lists, LISTS_MAX);
    TI_REQUIRE(n_areas >= 0 && n_moves >= 1 && (long long)n_moves * n_lists <= 8192, "beam reorder: %d moves in %d lists (at most 8192 in all)",
               n_moves, n_lists);
    if (n_areas == 0) return 0;
    ReorderArgs a = {};
    a.areas = static_cast<const Area*>(areas);
    a.n_areas = n_areas;
    a.n_lists = n_lists;
    a.n_moves = n_moves;
    a.moves = moves;
    a.status = ti_status_ptr();
    TI_REQUIRE(a.status != nullptr, "beam reorder: no status word");
    long long most = 0;
    for (int l = 0; l < n_lists; ++l) {
        a.first_area[l] = first_area[l];
        a.pieces[l] = pieces[l];
        most += pieces[l] * n_moves;
    }
    a.first_area[n_lists] = first_area[n_lists];
    const long long blocks = (most + RT / 32 - 1) / (RT / 32), room = (long long)BLOCKS * ti_sm_count();
    TI_CUDA(ti_launch(beam_reorder_kernel, dim3((unsigned)(blocks < room ? (blocks > 0 ? blocks : 1) : room)), dim3(RT),
                      (size_t)n_moves * n_lists * 4, stream, a));
    return 0;
}
