// Pages of the paged key/value caches of all layers: reserve, copy, fork, release, compact.
//
// One block table [B, max_blocks] (entries < 0: unassigned) and one array of reference counts [num_pages] (0: free) serve all
// layers; what a layer holds of a page lies in its own tensors (K and V codes or values, K and V scales), page-major, so that the
// first n slots of a page are one run of bytes in each.
//
// Every call is a plan by ONE block - it checks the whole call, picks the lowest free pages in order (so that results do not depend
// on timing) and either records an event and changes nothing, or updates counts and lists the moves (page, page, slots) - and, where
// data move, one kernel over the whole GPU that copies the listed runs and rewrites table rows.  Sources and destinations of one
// call are disjoint by construction (fork, compact) or checked (copy), so the moves are free of order.
//
// Plan: latency (num_pages counts are read twice, a warp per contiguous piece, ballots for the ranks): 4 to 8 us alone.  Moves: HBM, 2 bytes moved
// per byte copied: 400 MB in 57 us, 7 TB/s with what of it L2 still holds.
#include "common.cuh"

#include <algorithm>
#include <climits>
#include <tuple>
#include <type_traits>

namespace b200q {

B200Q_DEFINE_STATUS_WORD(pages_read_status)

namespace {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr int kMaxTensors = 256;          // per group of equal slot sizes and launch

// Workspace: header, moves, then what the plan needs.
struct Header {
    int32_t moves;      // listed moves
    int32_t ok;         // 0: the call was refused, nothing may change
    int32_t pad[2];
};
struct Move { int32_t src, dst, slots, pad; };

struct Tensors {        // two groups (codes or values, scales) of tensors with equal bytes per slot
    uint8_t* base[2][kMaxTensors];
    int64_t slot_bytes[2];
    int count[2];
    int page_size;
};

__device__ __forceinline__ void report(int event) { atomicMax(&g_device_status, event); }

// Exclusive prefix of one number per warp of the block, and their sum; `scratch`: kPlanWarps + 1 ints.  All threads call it.
__device__ __forceinline__ int warp_prefix(int mine, int* scratch, int* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) scratch[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        const int v = scratch[lane];
        int s = v;
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, s, o);
            if (lane >= o) s += u;
        }
        scratch[lane] = s - v;
        if (lane == 31) scratch[kPlanWarps] = s;
    }
    __syncthreads();
    *total = scratch[kPlanWarps];
    return scratch[warp];
}

// The pages a warp of the plan looks at: a contiguous piece, a multiple of 32 pages long.
struct Piece { int64_t lo, hi; };
__device__ __forceinline__ Piece warp_piece(int64_t n) {
    const int64_t per = ((n + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
    const int64_t lo = min(n, (int64_t)(threadIdx.x >> 5) * per);
    return {lo, min(n, lo + per)};
}

// Calls fn(page, rank) for the first `want` free pages in ascending order; returns how many free pages there are in all.
template <typename F> __device__ int visit_free(const int32_t* refs, int64_t n, int want, int* scratch, F fn) {
    const int lane = threadIdx.x & 31;
    const Piece piece = warp_piece(n);
    int mine = 0;
    for (int64_t i = piece.lo; i < piece.hi; i += 32) {
        const bool is_free = i + lane < piece.hi && refs[i + lane] <= 0;
        mine += __popc(__ballot_sync(0xFFFFFFFFu, is_free));
    }
    int total;
    int rank = warp_prefix(mine, scratch, &total);
    if (total >= want) {
        for (int64_t i = piece.lo; i < piece.hi && rank < want; i += 32) {
            const bool is_free = i + lane < piece.hi && refs[i + lane] <= 0;
            const unsigned b = __ballot_sync(0xFFFFFFFFu, is_free);
            const int r = rank + __popc(b & ((1u << lane) - 1u));
            if (is_free && r < want) fn((int)(i + lane), r);
            rank += __popc(b);
        }
    }
    return total;
}

// ---- reserve: pages for the next tokens of every sequence ---------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(int32_t* refs, int64_t num_pages, int32_t* table, const int32_t* lengths,
                                                               const int32_t* new_tokens, int uniform, int B, int max_blocks, int P,
                                                               int32_t* need_row, int32_t* need_block, int64_t need_cap, int32_t* row_first) {
    __shared__ int scratch[kPlanWarps + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    // blocks that the new tokens touch: [length / P, ceil((length + new) / P))
    auto blocks = [&](int b, int* lo, int* hi) {
        const int len = lengths[b], more = new_tokens ? new_tokens[b] : uniform;
        const int64_t end = ((int64_t)len + more + P - 1) / P;
        *lo = len / P;
        *hi = (int)min(end, (int64_t)max_blocks);
        if (more == 0) *hi = *lo;
        return len >= 0 && more >= 0 && (more == 0 || end <= max_blocks);
    };
    int64_t base = 0;                                 // pages needed by the rows before this round's
    int bad = 0;
    for (int b0 = 0; b0 < B; b0 += kPlanWarps) {
        const int b = b0 + warp;
        int count = 0;
        if (b < B) {
            int lo, hi;
            if (!blocks(b, &lo, &hi)) {
                bad = 1;
            } else {
                for (int j = lo; j < hi; j += 32) {
                    const bool open = j + lane < hi && table[(int64_t)b * max_blocks + j + lane] < 0;
                    count += __popc(__ballot_sync(0xFFFFFFFFu, open));
                }
            }
        }
        int total;
        const int before = warp_prefix(count, scratch, &total);
        if (b < B && lane == 0) row_first[b] = (int)(base + before);
        base += total;
        bad = __syncthreads_or(bad);
        if (bad || base > need_cap) break;            // uniform over the block; more than need_cap pages cannot be free
    }
    if (bad) {
        if (threadIdx.x == 0) report(EV_PAGE_CALL);
        return;
    }
    if (base > need_cap) {
        if (threadIdx.x == 0) report(EV_PAGES_EXHAUSTED);
        return;
    }
    for (int b = warp; b < B; b += kPlanWarps) {
        int lo, hi, k = row_first[b];
        blocks(b, &lo, &hi);
        for (int j = lo; j < hi; j += 32) {
            const bool open = j + lane < hi && table[(int64_t)b * max_blocks + j + lane] < 0;
            const unsigned m = __ballot_sync(0xFFFFFFFFu, open);
            if (open) {
                const int at = k + __popc(m & ((1u << lane) - 1u));
                need_row[at] = b;
                need_block[at] = j + lane;
            }
            k += __popc(m);
        }
    }
    __syncthreads();
    const int want = (int)base;
    const int have = visit_free(refs, num_pages, want, scratch, [&](int page, int k) {
        table[(int64_t)need_row[k] * max_blocks + need_block[k]] = page;
        refs[page] = 1;
    });
    if (have < want && threadIdx.x == 0) report(EV_PAGES_EXHAUSTED);
}

// ---- release: the pages of some sequences --------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) release_kernel(int32_t* refs, int64_t num_pages, int32_t* table, int32_t* lengths,
                                                      const int32_t* rows, int n, int B, int max_blocks) {
    __shared__ int seen;
    pdl_launch_dependents();
    pdl_wait();
    const int row = rows[blockIdx.x];
    if (row < 0) return;                               // padding
    if (row >= B) {
        if (threadIdx.x == 0) report(EV_PAGE_CALL);
        return;
    }
    if (threadIdx.x == 0) seen = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < (int)blockIdx.x; i += blockDim.x)
        if (rows[i] == row) seen = 1;                  // the first of equal rows releases it
    __syncthreads();
    if (seen) return;
    for (int j = threadIdx.x; j < max_blocks; j += blockDim.x) {
        int32_t* entry = table + (int64_t)row * max_blocks + j;
        const int page = *entry;
        *entry = -1;
        if (page < 0) continue;
        if (page >= num_pages || atomicSub(refs + page, 1) <= 0) {      // a page that nobody held: its count stays
            if (page < num_pages) atomicAdd(refs + page, 1);
            report(EV_PAGE_CALL);
        }
    }
    if (threadIdx.x == 0) lengths[row] = 0;
}

// ---- copy: listed pairs of pages -----------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) copy_plan_kernel(const int32_t* src, const int32_t* dst, int n, int64_t num_pages, int P,
                                                                 Header* header, Move* moves, int32_t* mark) {
    __shared__ int bad;
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x == 0) bad = 0;
    for (int64_t i = threadIdx.x; i < num_pages; i += kPlanThreads) mark[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int s = src[i], d = dst[i];
        const bool skip = s < 0 || d < 0;
        moves[i] = {s, d, skip ? 0 : P, 0};
        if (skip) continue;
        if (s >= num_pages || d >= num_pages || atomicAdd(mark + d, 1) != 0) bad = 1;      // out of range, or two copies into one page
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int s = src[i];
        if (moves[i].slots > 0 && s < num_pages && mark[s] != 0) bad = 1;                  // a source that is copied over
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (bad) report(EV_PAGE_CALL);
        *header = {bad ? 0 : n, bad ? 0 : 1, {0, 0}};
    }
}

// ---- fork: sequences that continue others --------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(int32_t* refs, int64_t num_pages, int32_t* table, int32_t* lengths,
                                                                 const int32_t* parents, const int32_t* children, int n, int B, int max_blocks,
                                                                 int P, Header* header, Move* moves, int32_t* is_child) {
    __shared__ int scratch[kPlanWarps + 1];
    __shared__ int bad;
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x == 0) bad = 0;
    for (int b = threadIdx.x; b < B; b += kPlanThreads) is_child[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int p = parents[i], c = children[i];
        if (p < 0 || c < 0) continue;                                   // padding
        if (p >= B || c >= B || atomicAdd(is_child + c, 1) != 0) bad = 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int p = parents[i], c = children[i];
        if (p < 0 || c < 0 || p >= B || c >= B) continue;
        const int len = lengths[p];
        if (is_child[p] != 0 || len < 0 || len > (int64_t)max_blocks * P || lengths[c] != 0) bad = 1;
    }
    // a child's row must be empty: whoever overwrote it would lose its pages.  A warp per child.
    for (int i = threadIdx.x >> 5; i < n; i += kPlanWarps) {
        const int p = parents[i], c = children[i];
        if (p < 0 || c < 0 || c >= B) continue;
        bool held = false;
        for (int j = lane; j < max_blocks; j += 32) held |= table[(int64_t)c * max_blocks + j] >= 0;
        if (held) bad = 1;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) {
            report(EV_PAGE_CALL);
            *header = {0, 0, {0, 0}};
        }
        return;
    }
    // the last page of a parent that is not full is copied: its slots may differ from now on
    int want = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        int src = -1, rest = 0;
        if (i < n && parents[i] >= 0 && children[i] >= 0) {
            const int len = lengths[parents[i]];
            rest = len % P;
            if (rest > 0) src = table[(int64_t)parents[i] * max_blocks + len / P];
            if (src >= num_pages) src = -1;
        }
        const unsigned b = __ballot_sync(0xFFFFFFFFu, src >= 0);
        int total;
        const int before = warp_prefix(__popc(b), scratch, &total);
        if (src >= 0) moves[want + before + __popc(b & ((1u << lane) - 1u))] = {src, -1, rest, i};
        want += total;
    }
    __syncthreads();
    const int have = visit_free(refs, num_pages, want, scratch, [&](int page, int k) {
        const int i = moves[k].pad;
        moves[k].dst = page;
        refs[page] = 1;
        table[(int64_t)children[i] * max_blocks + lengths[parents[i]] / P] = page;
    });
    __syncthreads();
    const bool ok = have >= want;
    for (int i = threadIdx.x; ok && i < n; i += kPlanThreads)
        if (parents[i] >= 0 && children[i] >= 0) lengths[children[i]] = lengths[parents[i]];
    if (threadIdx.x == 0) {
        if (!ok) report(EV_PAGES_EXHAUSTED);
        *header = {ok ? want : 0, ok ? 1 : 0, {0, 0}};
    }
}

// ---- compact: live pages to the low end ----------------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(int32_t* refs, int64_t num_pages, int P, Header* header, Move* moves,
                                                                    int32_t* remap) {
    __shared__ int scratch[kPlanWarps + 1];
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    const Piece piece = warp_piece(num_pages);
    int mine = 0;
    for (int64_t i = piece.lo; i < piece.hi; i += 32)
        mine += __popc(__ballot_sync(0xFFFFFFFFu, i + lane < piece.hi && refs[i + lane] > 0));
    int live;
    warp_prefix(mine, scratch, &live);
    // the k-th free page below `live` takes the k-th live page at or above it
    int free_below = 0, live_above = 0;
    for (int64_t i = piece.lo; i < piece.hi; i += 32) {
        const int64_t page = i + lane;
        const bool in = page < piece.hi, is_live = in && refs[page] > 0;
        free_below += __popc(__ballot_sync(0xFFFFFFFFu, in && !is_live && page < live));
        live_above += __popc(__ballot_sync(0xFFFFFFFFu, is_live && page >= live));
    }
    int moved, same;
    int hole = warp_prefix(free_below, scratch, &moved), mover = warp_prefix(live_above, scratch, &same);
    for (int64_t i = piece.lo; i < piece.hi; i += 32) {
        const int64_t page = i + lane;
        const bool in = page < piece.hi, is_live = in && refs[page] > 0;
        const unsigned h = __ballot_sync(0xFFFFFFFFu, in && !is_live && page < live), m = __ballot_sync(0xFFFFFFFFu, is_live && page >= live);
        const unsigned below = (1u << lane) - 1u;
        if (h >> lane & 1u) moves[hole + __popc(h & below)].dst = (int)page;
        if (m >> lane & 1u) {
            Move& mv = moves[mover + __popc(m & below)];
            mv.src = (int)page;
            mv.slots = P;
        }
        if (in) remap[page] = is_live ? (int)page : -1;
        hole += __popc(h);
        mover += __popc(m);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < moved; k += kPlanThreads) {
        const Move mv = moves[k];
        remap[mv.src] = mv.dst;
        refs[mv.dst] = refs[mv.src];
        refs[mv.src] = 0;
    }
    if (threadIdx.x == 0) *header = {moved, 1, {0, 0}};
}

// ---- the moves, and the rows of the table --------------------------------------------------------------------------------
// What a warp copies at a time: kBatch loads of a unit per lane, all in flight.
constexpr int kBatch = 4;
template <typename U> __device__ __forceinline__ void copy_run(uint8_t* dst, const uint8_t* src, int64_t bytes) {
    const int lane = threadIdx.x & 31;
    const int64_t n = bytes / (int64_t)sizeof(U);
    U v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
        if (lane + 32 * j < n) v[j] = __ldcs(reinterpret_cast<const U*>(src) + lane + 32 * j);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
        if (lane + 32 * j < n) reinterpret_cast<U*>(dst)[lane + 32 * j] = v[j];
}

struct RowWork {                     // table rows that the kernel rewrites beside the copies
    int32_t* table;
    int32_t* refs;
    const int32_t* lengths;          // fork
    const int32_t* parents;
    const int32_t* children;
    const int32_t* remap;            // compact
    int rows, max_blocks;            // rows: pairs (fork) or sequences (compact); 0: none
    int64_t num_pages;
};

template <typename U>
__global__ void __launch_bounds__(256) move_kernel(const __grid_constant__ Tensors t, const Header* header, const Move* moves, int64_t pieces0,
                                                   int64_t pieces1, const __grid_constant__ RowWork r) {
    pdl_launch_dependents();
    pdl_wait();
    if (header->ok == 0) return;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5), first = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    constexpr int64_t kRunBytes = 32 * kBatch * sizeof(U);
    // pieces of a move: those of the first group's tensors, then the second's
    const int64_t in0 = pieces0 * t.count[0], per_move = in0 + pieces1 * t.count[1], total = per_move * header->moves;
    for (int64_t it = first; it < total; it += warps) {
        const int64_t k = it / per_move;
        int64_t rest = it - k * per_move;
        const int g = rest >= in0;
        if (g) rest -= in0;
        const int64_t pieces = g ? pieces1 : pieces0;
        const int i = (int)(rest / pieces);
        const int64_t off = (rest - i * pieces) * kRunBytes;
        const Move m = moves[k];
        const int64_t bytes = m.slots * t.slot_bytes[g] - off, page_bytes = t.page_size * t.slot_bytes[g];
        if (bytes <= 0) continue;
        uint8_t* base = t.base[g][i];
        copy_run<U>(base + m.dst * page_bytes + off, base + m.src * page_bytes + off, min(bytes, kRunBytes));
    }
    if (r.rows == 0) return;
    const int64_t strips = (r.max_blocks + 31) / 32, row_items = r.rows * strips;
    for (int64_t it = first; it < row_items; it += warps) {
        const int64_t i = it / strips;
        const int64_t j = (it - i * strips) * 32 + lane;
        if (j >= r.max_blocks) continue;
        if (r.remap != nullptr) {
            int32_t* entry = r.table + i * r.max_blocks + j;
            const int page = *entry;
            if (page >= 0 && page < r.num_pages) {
                const int now = r.remap[page];
                if (now >= 0 && now != page) *entry = now;
            }
        } else {
            const int p = r.parents[i], c = r.children[i];
            if (p < 0 || c < 0 || j >= r.lengths[p] / t.page_size) continue;
            const int page = r.table[(int64_t)p * r.max_blocks + j];
            if (page < 0) continue;
            r.table[(int64_t)c * r.max_blocks + j] = page;
            if (page < r.num_pages) atomicAdd(r.refs + page, 1);
        }
    }
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

cudaError_t launch_pdl(cudaStream_t stream, int blocks, int threads, const void* kernel, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tuning_get("no_pdl") ? 0 : 1;
    return cudaLaunchKernelExC(&cfg, kernel, args);
}
template <typename... P, typename... A>
int launch(cudaStream_t stream, int64_t blocks, int threads, void (*kernel)(P...), A... a) {
    std::tuple<std::decay_t<P>...> values(a...);
    return std::apply(
        [&](auto&... v) {
            void* args[] = {(void*)&v...};
            return launch_pdl(stream, (int)blocks, threads, (const void*)kernel, args) == cudaSuccess ? finish_launch() : B200Q_ERR_LAUNCH;
        },
        values);
}

// Tensors of the caches, [n0] with slot0 bytes per slot and [n1] with slot1, moved as the list says; `r` once.
int run_moves(void* const* bases0, int n0, int64_t slot0, void* const* bases1, int n1, int64_t slot1, int P, const Header* header,
              const Move* moves, RowWork r, cudaStream_t stream) {
    uintptr_t bits = (uintptr_t)slot0 | (uintptr_t)(n1 ? slot1 : 0);
    for (int i = 0; i < n0; ++i) bits |= (uintptr_t)bases0[i];
    for (int i = 0; i < n1; ++i) bits |= (uintptr_t)bases1[i];
    for (int at = 0; at == 0 || at < std::max(n0, n1); at += kMaxTensors) {
        Tensors t = {};
        t.count[0] = std::max(0, std::min(kMaxTensors, n0 - at));
        t.count[1] = std::max(0, std::min(kMaxTensors, n1 - at));
        for (int i = 0; i < t.count[0]; ++i) t.base[0][i] = (uint8_t*)bases0[at + i];
        for (int i = 0; i < t.count[1]; ++i) t.base[1][i] = (uint8_t*)bases1[at + i];
        t.slot_bytes[0] = slot0;
        t.slot_bytes[1] = n1 ? slot1 : 0;
        t.page_size = P;
        const int unit = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
        const int64_t run = 32 * kBatch * unit, pieces0 = (P * slot0 + run - 1) / run, pieces1 = n1 ? (P * slot1 + run - 1) / run : 1;
        const int64_t blocks = (int64_t)sm_count() * 8;
        const int rc = unit == 16 ? launch(stream, blocks, 256, move_kernel<uint4>, t, header, moves, pieces0, pieces1, r)
                     : unit == 4  ? launch(stream, blocks, 256, move_kernel<uint32_t>, t, header, moves, pieces0, pieces1, r)
                                  : launch(stream, blocks, 256, move_kernel<uint8_t>, t, header, moves, pieces0, pieces1, r);
        if (rc != B200Q_OK) return rc;
        r.rows = 0;
    }
    return B200Q_OK;
}

constexpr int kMaxBlocks = 1 << 24;      // of a sequence: a round of the reserve plan counts 32 rows in 32 bits

bool bad_tensors(void* const* bases0, int n0, int64_t slot0, void* const* bases1, int n1, int64_t slot1) {
    if (n0 < 0 || n1 < 0 || (n0 > 0 && (bases0 == nullptr || slot0 <= 0)) || (n1 > 0 && (bases1 == nullptr || slot1 <= 0))) return true;
    for (int i = 0; i < n0; ++i)
        if (bases0[i] == nullptr) return true;
    for (int i = 0; i < n1; ++i)
        if (bases1[i] == nullptr) return true;
    return false;
}

}  // namespace

// bytes: header, moves (up to `moves`), then `ints` int32
static size_t workspace(int64_t moves, int64_t ints) { return sizeof(Header) + sizeof(Move) * (size_t)moves + round16(4 * (size_t)ints); }

size_t reserve_workspace_impl(int B, int64_t num_pages) { return B <= 0 || num_pages <= 0 ? 0 : round16(4 * (2 * (size_t)num_pages + B)); }
size_t copy_workspace_impl(int n, int64_t num_pages) { return n <= 0 || num_pages <= 0 ? 0 : workspace(n, num_pages); }
size_t fork_workspace_impl(int n, int B) { return n <= 0 || B <= 0 ? 0 : workspace(n, B); }
size_t compact_workspace_impl(int64_t num_pages) { return num_pages <= 0 ? 0 : workspace((num_pages + 1) / 2, 0); }

int reserve_pages_impl(int32_t* refs, int64_t num_pages, int32_t* table, const int32_t* lengths, const int32_t* new_tokens, int uniform,
                       int B, int max_blocks, int page_size, void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (refs == nullptr || table == nullptr || lengths == nullptr) return B200Q_ERR_BAD_ARG;
    if (num_pages <= 0 || num_pages > INT32_MAX || B <= 0 || max_blocks <= 0 || page_size <= 0 || (new_tokens == nullptr && uniform < 0))
        return B200Q_ERR_BAD_ARG;
    if (max_blocks > kMaxBlocks) return B200Q_ERR_UNSUPPORTED;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < reserve_workspace_impl(B, num_pages)) return B200Q_ERR_WORKSPACE;
    int32_t* need_row = (int32_t*)ws;
    return launch(stream, 1, kPlanThreads, reserve_kernel, refs, num_pages, table, lengths, new_tokens, uniform, B, max_blocks, page_size,
                  need_row, need_row + num_pages, num_pages, need_row + 2 * num_pages);
}

int release_sequences_impl(int32_t* refs, int64_t num_pages, int32_t* table, int32_t* lengths, const int32_t* rows, int n, int B,
                           int max_blocks, cudaStream_t stream) {
    if (refs == nullptr || table == nullptr || lengths == nullptr || rows == nullptr) return B200Q_ERR_BAD_ARG;
    if (num_pages <= 0 || num_pages > INT32_MAX || n <= 0 || B <= 0 || max_blocks <= 0) return B200Q_ERR_BAD_ARG;
    return launch(stream, n, 128, release_kernel, refs, num_pages, table, lengths, rows, n, B, max_blocks);
}

int copy_pages_impl(void* const* bases0, int n0, int64_t slot0, void* const* bases1, int n1, int64_t slot1, const int32_t* src,
                    const int32_t* dst, int n, int64_t num_pages, int page_size, void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (bad_tensors(bases0, n0, slot0, bases1, n1, slot1) || src == nullptr || dst == nullptr) return B200Q_ERR_BAD_ARG;
    if (num_pages <= 0 || num_pages > INT32_MAX || n <= 0 || page_size <= 0) return B200Q_ERR_BAD_ARG;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < copy_workspace_impl(n, num_pages)) return B200Q_ERR_WORKSPACE;
    Header* header = (Header*)ws;
    Move* moves = (Move*)(header + 1);
    const int rc = launch(stream, 1, kPlanThreads, copy_plan_kernel, src, dst, n, num_pages, page_size, header, moves, (int32_t*)(moves + n));
    return rc != B200Q_OK ? rc : run_moves(bases0, n0, slot0, bases1, n1, slot1, page_size, header, moves, RowWork{}, stream);
}

int fork_sequences_impl(void* const* bases0, int n0, int64_t slot0, void* const* bases1, int n1, int64_t slot1, int32_t* refs,
                        int64_t num_pages, int32_t* table, int32_t* lengths, const int32_t* parents, const int32_t* children, int n, int B,
                        int max_blocks, int page_size, void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (bad_tensors(bases0, n0, slot0, bases1, n1, slot1) || refs == nullptr || table == nullptr || lengths == nullptr || parents == nullptr ||
        children == nullptr)
        return B200Q_ERR_BAD_ARG;
    if (num_pages <= 0 || num_pages > INT32_MAX || n <= 0 || B <= 0 || max_blocks <= 0 || page_size <= 0) return B200Q_ERR_BAD_ARG;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < fork_workspace_impl(n, B)) return B200Q_ERR_WORKSPACE;
    Header* header = (Header*)ws;
    Move* moves = (Move*)(header + 1);
    const int rc = launch(stream, 1, kPlanThreads, fork_plan_kernel, refs, num_pages, table, lengths, parents, children, n, B, max_blocks,
                          page_size, header, moves, (int32_t*)(moves + n));
    if (rc != B200Q_OK) return rc;
    const RowWork r = {table, refs, lengths, parents, children, nullptr, n, max_blocks, num_pages};
    return run_moves(bases0, n0, slot0, bases1, n1, slot1, page_size, header, moves, r, stream);
}

int compact_pages_impl(void* const* bases0, int n0, int64_t slot0, void* const* bases1, int n1, int64_t slot1, int32_t* refs,
                       int64_t num_pages, int32_t* table, int B, int max_blocks, int page_size, int32_t* remap, void* ws, size_t ws_bytes,
                       cudaStream_t stream) {
    if (bad_tensors(bases0, n0, slot0, bases1, n1, slot1) || refs == nullptr || table == nullptr || remap == nullptr) return B200Q_ERR_BAD_ARG;
    if (num_pages <= 0 || num_pages > INT32_MAX || B <= 0 || max_blocks <= 0 || page_size <= 0) return B200Q_ERR_BAD_ARG;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < compact_workspace_impl(num_pages)) return B200Q_ERR_WORKSPACE;
    Header* header = (Header*)ws;
    Move* moves = (Move*)(header + 1);
    const int rc = launch(stream, 1, kPlanThreads, compact_plan_kernel, refs, num_pages, page_size, header, moves, remap);
    if (rc != B200Q_OK) return rc;
    const RowWork r = {table, refs, nullptr, nullptr, nullptr, remap, B, max_blocks, num_pages};
    return run_moves(bases0, n0, slot0, bases1, n1, slot1, page_size, header, moves, r, stream);
}

}  // namespace b200q
