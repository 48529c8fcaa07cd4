// Low-rank adapters of many requests beside one shared projection.
//
//   out[t] = cast(y[t] + s[l] * B[l] (A[l] x[t])),   l = ids[t];   ids[t] < 0: out[t] = y[t]
//
// A [L, R, K] and B [L, N, R] hold the factors of L adapters, of which adapter l uses the first ranks[l] of R; x [rows, K], y and out
// [rows, N] (out may be y).  Products are summed in fp32, the R values between the factors stay in fp32 (or in as many bits), and the
// sum with y is rounded once.
//
// One launch for both products: a thread-block cluster per adapter and up to 16 of the rows that use it.  Rows are looked at in windows of 256,
// in which every CTA finds the groups; the clusters of a window take them in turn, or, when there are more of them than groups, slices of a
// group's columns.  The CTAs of a cluster cut K: every warp multiplies its pieces of the rows with the factor A on mma.sync, straight from
// global memory - the order of the summands is free, so a lane takes 16 contiguous bytes of a row as the k indices of two instructions.
// The partial sums meet in shared memory, then through distributed shared memory in every CTA; then the CTAs cut N: 32 columns per warp
// and round, a lane with contiguous bytes of B again and 16 bytes of y, the next rounds' loads in flight during this one's products.  The
// values between the factors enter the second product as two 16-bit terms, scaled by a power of two per row, which holds them to about 2^-21.
//
// Beside a projection of a few rows and small ranks none of this runs: the integer matvec takes the adapters along (lora_qmatvec_impl below).
//
// Bound by latency for a few rows (a chain of ids, first factor, two meetings, second factor: 5.9 us for one row of rank 16, 4096 x 4096, and
// 13.5 for 32 rows of 24 adapters of rank 64, 6144 x 4096, 1.8 TB/s), by L2 and the products for prompts, whose groups of 16 rows read both factors
// again (512 rows of rank 64, 14336 x 4096: 30 us).
#include "gemv_params.cuh"

#include <algorithm>
#include <type_traits>

namespace b200q {

B200Q_DEFINE_STATUS_WORD(lora_read_status)

int qmatvec_impl(int bits, const void* x, const uint8_t* codes, const void* scales, const void* zeros,
                 const void* residual, void* y, int B, int64_t N, int64_t K, int group_size, int act_dtype,
                 int scale_dtype, const void* residual_in, const void* norm_weight, int norm_w_dtype, float eps,
                 void* z_out, void* normed_out, cudaStream_t stream, const float* add32);
int lora_rows_qmatvec(int bits, const void* x, const uint8_t* codes, const void* scales, const void* zeros, const void* residual, void* y, int B,
                      int64_t N, int64_t K, int group_size, int act_dtype, int scale_dtype, const LoraRows& lora, cudaStream_t stream);

namespace {

struct LoraParams {
    const void* x;            // [rows, K]
    const void* y;            // [rows, N] or null: 0
    void* out;                // [rows, N], in the rows' type or (out32) fp32
    const void* a;            // [L, R, K]
    const void* b;            // [L, N, R]
    const float* scaling;     // [L] or null: 1
    const int32_t* ranks;     // [L] or null: R
    const int32_t* ids;       // [rows]
    float* low;               // [rows, R] scratch of the general kernels
    int64_t rows, K, N;
    int L, R, out32;
};

// Adapter of a row, or -1.  (Both past the L1: the cluster kernel also reads them while the kernel before may still write them.)
__device__ __forceinline__ int adapter_of(const LoraParams& p, int64_t row) {
    const int id = __ldcg(p.ids + row);
    return id < p.L ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraParams& p, int id) { return p.ranks ? max(0, min(p.R, __ldcg(p.ranks + id))) : p.R; }

// ---- any size: a warp per value between the factors, then a thread per result ------------------------------------------------
template <typename T> __global__ void __launch_bounds__(256) lora_shrink_any_kernel(const __grid_constant__ LoraParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5), items = p.rows * p.R;
    for (int64_t it = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t row = it / p.R;
        const int r = (int)(it - row * p.R), id = adapter_of(p, row);
        if (lane == 0 && r == 0 && p.ids[row] >= p.L) atomicMax(&g_device_status, (int)EV_LORA_ADAPTER);
        if (id < 0 || r >= rank_of(p, id)) continue;
        const T* x = reinterpret_cast<const T*>(p.x) + row * p.K;
        const T* a = reinterpret_cast<const T*>(p.a) + ((int64_t)id * p.R + r) * p.K;
        float s = 0.0f;
        for (int64_t k = lane; k < p.K; k += 32) s = fmaf(to_f32(x[k]), to_f32(a[k]), s);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (lane == 0) p.low[it] = s;
    }
}
template <typename T> __global__ void __launch_bounds__(256) lora_expand_any_kernel(const __grid_constant__ LoraParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t threads = (int64_t)gridDim.x * blockDim.x, items = p.rows * p.N;
    for (int64_t it = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; it < items; it += threads) {
        const int64_t row = it / p.N, n = it - row * p.N;
        const int id = adapter_of(p, row);
        const T y = p.y ? reinterpret_cast<const T*>(p.y)[it] : from_f32<T>(0.0f);
        float s = 0.0f;
        if (id >= 0) {
            const T* b = reinterpret_cast<const T*>(p.b) + ((int64_t)id * p.N + n) * p.R;
            const float* low = p.low + row * p.R;
            const int rank = rank_of(p, id);
            for (int r = 0; r < rank; ++r) s = fmaf(to_f32(b[r]), low[r], s);
            if (p.scaling) s *= p.scaling[id];
        }
        if (p.out32) reinterpret_cast<float*>(p.out)[it] = id < 0 ? to_f32(y) : to_f32(y) + s;
        else reinterpret_cast<T*>(p.out)[it] = id < 0 ? y : from_f32<T>(to_f32(y) + s);
    }
}

template <typename F> int launch(F kernel, int64_t blocks, int threads, cudaStream_t stream, const LoraParams& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tuning_get("no_pdl") ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? finish_launch() : B200Q_ERR_LAUNCH;
}

template <typename T> int any_size(const LoraParams& p, cudaStream_t stream) {
    const int64_t cap = (int64_t)sm_count() * 8;
    const int rc = launch(lora_shrink_any_kernel<T>, std::min(cap, (p.rows * p.R + 7) / 8), 256, stream, p);
    return rc != B200Q_OK ? rc : launch(lora_expand_any_kernel<T>, std::min(cap, (p.rows * p.N + 255) / 256), 256, stream, p);
}

// ---- the cluster kernel: K a multiple of 8, R a multiple of 4 up to 256, 16-byte aligned factors and rows ------------------------
constexpr int kRows = 16, kMaxRank = 256, kRankBlock = 64;
constexpr int kGather = 16;               // CTAs whose sums are fetched at a time (8: 0.6 us longer with 16 CTAs)
constexpr int kWindow = 256;              // rows that one group may come from

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float load_remote(const float* local, uint32_t cta) {
    uint32_t addr;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
// 16 bytes into shared memory behind the thread's back, or zeros
__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const __half*) {
    mma_m16n8k16(d, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const __nv_bfloat16*) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// zeros for all but the first n (> 0 or not) values of a piece
__device__ __forceinline__ uint32_t keep2(uint32_t v, int n) { return n >= 2 ? v : n == 1 ? v & 0xFFFFu : 0u; }
__device__ __forceinline__ void keep_ranks(uint2& v, int n) {
    v.x = keep2(v.x, n);
    v.y = keep2(v.y, n - 2);
}
__device__ __forceinline__ void keep_ranks(uint4& v, int n) {
    v.x = keep2(v.x, n);
    v.y = keep2(v.y, n - 2);
    v.z = keep2(v.z, n - 4);
    v.w = keep2(v.w, n - 6);
}

// shared memory: partial sums of the warps, of the CTA, and the two terms of the rows between the factors
struct LoraSmem {
    int low_stride;           // 16-bit values per row of a term: the rank in whole steps of 32, and 8 against bank conflicts
    size_t part, cta, hi, lo, ring, bytes;
};
__host__ __device__ inline LoraSmem lora_smem(int R, int warps, int depth) {
    LoraSmem s;
    const int block = R < kRankBlock ? (R + 7) / 8 * 8 : kRankBlock;
    s.low_stride = (R + 31) / 32 * 32 + 8;
    s.part = 0;
    s.cta = s.part + sizeof(float) * warps * kRows * block;
    s.hi = s.cta + sizeof(float) * kRows * ((R + 7) / 8 * 8);
    s.lo = s.hi + 2 * (size_t)kRows * s.low_stride;
    s.ring = s.lo + 2 * (size_t)kRows * s.low_stride;
    s.bytes = s.ring + sizeof(uint4) * 32 * 4 * depth * warps;
    return s;
}

// NT: rank tiles of 8 that a warp accumulates at a time.  NT 2 takes ranks by 16 (8 bytes of B per lane), NT 4 and 8 by 32 (16 bytes).
// For these two rounds of B are in flight in a ring of shared memory, from before the products with A on (NT 2: one, in registers).  32 and 512
// rows of rank 64, fp16, with a projection 6144 x 4096: 22.5 -> 21.5 us, 68.4 -> 66.8; three or four rounds ahead: 21.8, 22.1 and 67.2.
constexpr int ring_depth(int NT) { return NT <= 2 ? 0 : 2; }
// SLICED: several clusters may take slices of a group's columns (a template parameter: one row 10.9 us against 11.3 with the choice at run time).
template <typename T, int NT, int kWarps, bool SLICED>
__global__ void __launch_bounds__(kWarps * 32, 2) lora_cluster_kernel(const __grid_constant__ LoraParams p, int per_window, int max_slices, int vector_rows) {
    using Piece = std::conditional_t<NT <= 2, uint2, uint4>;
    constexpr int kPer = sizeof(Piece) / 2;                  // ranks in a lane's piece
    constexpr int kStep = 4 * kPer;                          // ranks of a round
    constexpr int DEPTH = ring_depth(NT);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float row_scale[kRows];
    __shared__ __align__(16) int id_of[kWindow];             // -1: none, -2: no such row
    __shared__ int before_of[kWindow];                       // rows of the same adapter ahead of a row in the window
    __shared__ int leaders[kWindow];
    __shared__ int leads[kWarps];
    __shared__ int row_of[kRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t cta = cluster_rank(), ctas = cluster_size();
    const LoraSmem at = lora_smem(p.R, kWarps, DEPTH);
    float* part = reinterpret_cast<float*>(smem + at.part);
    float* own = reinterpret_cast<float*>(smem + at.cta);
    T* hi = reinterpret_cast<T*>(smem + at.hi);
    T* lo = reinterpret_cast<T*>(smem + at.lo);
    const T* y = reinterpret_cast<const T*>(p.y);
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    const int K = (int)p.K, N = (int)p.N;                    // below 2^30
    const int chunks = (K + 31) / 32, per = (chunks + (int)ctas - 1) / (int)ctas;
    const int c_lo = min(chunks, (int)cta * per), c_hi = min(chunks, c_lo + per);
    const int strips = (N + 31) / 32;
    pdl_launch_dependents();

    // ---- the window's groups: every sixteenth row of an adapter leads one ----
    const int cluster = (int)(blockIdx.x / ctas), window = cluster / per_window, turn = cluster - window * per_window;
    const int64_t row0 = (int64_t)window * kWindow;
    const bool looks = kWarps * 32 <= kWindow || threadIdx.x < kWindow;
    int my_id, before, groups, slices;
    auto read_id = [&]() { return looks && row0 + threadIdx.x < p.rows ? max(adapter_of(p, row0 + threadIdx.x), -1) : -2; };
    auto find_groups = [&]() {
        if (looks) id_of[threadIdx.x] = my_id;
        __syncthreads();
        before = 0;
        for (int i = 0; my_id > -2 && i < (int)threadIdx.x / 4; ++i) {
            const int4 v = reinterpret_cast<const int4*>(id_of)[i];
            before += (v.x == my_id) + (v.y == my_id) + (v.z == my_id) + (v.w == my_id);
        }
        for (int i = threadIdx.x / 4 * 4; my_id > -2 && i < (int)threadIdx.x; ++i) before += id_of[i] == my_id;
        if (looks) before_of[threadIdx.x] = before;
        const unsigned lead_vote = __ballot_sync(0xFFFFFFFFu, my_id > -2 && before % kRows == 0);
        if (lane == 0) leads[warp] = __popc(lead_vote);
        __syncthreads();
        int my_place = __popc(lead_vote & ((1u << lane) - 1u));
        groups = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            if (i < warp) my_place += leads[i];
            groups += leads[i];
        }
        if (lead_vote >> lane & 1u) leaders[my_place] = threadIdx.x;
        // fewer groups than clusters: several clusters take slices of a group's columns, and all of its products with A
        slices = SLICED && groups > 0 && 2 * groups <= per_window ? min(per_window / groups, max_slices) : 1;
        __syncthreads();
    };
    // While the kernel before ends, the groups are found from what ids and ranks say now, and the CTA's slices of the first group's
    // factors are brought into L2.  All of it is a guess: whatever counts is read again behind the wait.
    my_id = read_id();
    find_groups();
    if (turn < groups * slices) {
        const int slice = SLICED && slices > 1 ? turn / groups : 0;
        const int id = id_of[leaders[turn - slice * groups]], rank = id < 0 ? 0 : rank_of(p, id);
        const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)max(id, 0) * p.R * p.K;
        const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)max(id, 0) * p.N * p.R;
        const int lines = (c_hi - c_lo + 1) / 2;
        for (int i = threadIdx.x; i < rank * lines; i += kWarps * 32) {
            const int r = i / lines;
            prefetch_l2(a + (int64_t)r * K + c_lo * 32 + (i - r * lines) * 64);
        }
        const int strip_lines = (p.R * 64 + 127) / 128;
        for (int s = (slice * (int)ctas + (int)cta) * kWarps + warp; rank > 0 && s < strips; s += slices * (int)ctas * kWarps)
            for (int i = lane; i < strip_lines; i += 32)
                if ((int64_t)s * 32 * p.R + i * 64 < (int64_t)N * p.R) prefetch_l2(b + (int64_t)s * 32 * p.R + i * 64);
    }
    pdl_wait();
    const int id_now = read_id();
    if (__syncthreads_or(id_now != my_id)) {
        my_id = id_now;
        find_groups();
    }

    for (int item = turn; item < groups * slices; item += per_window) {      // all CTAs of a cluster agree
        const int slice = SLICED && slices > 1 ? item / groups : 0, s_first = (slice * (int)ctas + (int)cta) * kWarps + warp, s_step = slices * (int)ctas * kWarps;
        const int lead = leaders[item - slice * groups], id = id_of[lead], ahead = before_of[lead];
        if (threadIdx.x < kRows) row_of[threadIdx.x] = -1;
        __syncthreads();
        if (my_id == id && before >= ahead && before < ahead + kRows) row_of[before - ahead] = threadIdx.x;
        const int rank = id < 0 ? 0 : rank_of(p, id);
        const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)max(id, 0) * p.R * p.K;
        const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)max(id, 0) * p.N * p.R;
        __syncthreads();
        if (id < 0) {
            if (cta == 0 && threadIdx.x < kRows && row_of[threadIdx.x] >= 0 && p.ids[row0 + row_of[threadIdx.x]] >= p.L)
                atomicMax(&g_device_status, (int)EV_LORA_ADAPTER);
            if (p.out == p.y) {
                __syncthreads();
                continue;
            }
        }
        const int rank8 = (rank + 7) / 8 * 8, rank16 = (rank + 15) / 16 * 16;
        const int t0 = row_of[g], t1 = row_of[g + 8];
        const bool r0 = t0 >= 0, r1 = t1 >= 0;

        // a round's loads of B, a lane's piece for each of four instructions: j's column n is 32 s + 8 (n / 2) + 2 j + n % 2, so that a
        // lane's results are columns 32 s + 8 q .. + 7 of rows g and g + 8
        const int first_col = (g >> 1) * 8 + (g & 1), b_next = 2 * p.R;
        const T* b_lane = b + (int64_t)(s_first * 32 + first_col) * p.R + q * kPer;
        const int64_t b_step = (int64_t)s_step * 32 * p.R;
        const bool ragged = rank % kPer != 0;
        auto load_b = [&](Piece (&w)[4], const T* from, int s, int k0) {
            const int k = k0 + q * kPer;
            const bool whole = s * 32 + 32 <= N;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = {};
                if (k < rank && (whole || s * 32 + first_col + 2 * j < N)) w[j] = __ldg(reinterpret_cast<const Piece*>(from + j * b_next + k0));
            }
            if (ragged && k < rank && k + kPer > rank)       // values behind the rank are not the adapter's
#pragma unroll
                for (int j = 0; j < 4; ++j) keep_ranks(w[j], rank - k);
        };
        Piece w[4];
        // the ring: a lane copies its pieces of the rounds ahead and reads them back itself, so that nothing but its own copies is waited for
        uint4* ring = reinterpret_cast<uint4*>(smem + at.ring) + warp * (DEPTH * 4 * 32) + lane;
        const T* ring_b = b_lane;
        int ring_s = s_first, ring_k = 0, ring_at = 0;
        auto copy_round = [&]() {                            // of the round that ring_s and ring_k are at; into the slot that was read last
            if (ring_s < strips && rank > 0) {
                const bool in = ring_k + q * kPer < rank;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool live = in && ring_s * 32 + first_col + 2 * j < N;
                    cp_async16_or_zero(ring + (ring_at * 4 + j) * 32, live ? ring_b + j * b_next + ring_k : b, live);
                }
                ring_k += kStep;
                if (ring_k >= rank) {
                    ring_k = 0;
                    ring_s += s_step;
                    ring_b += b_step;
                }
            }
            cp_async_commit();
            if (++ring_at == DEPTH) ring_at = 0;
        };
        if constexpr (DEPTH > 0) {
            for (int i = 0; i < DEPTH; ++i) copy_round();
        } else {
            load_b(w, b_lane, s_first, 0);
        }

        // ---- rows times A: the CTA's chunks of 32 k, dealt to its warps; a lane holds k = 8q .. 8q + 7 of a chunk ----
        const T* x0 = reinterpret_cast<const T*>(p.x) + (row0 + max(t0, 0)) * p.K + q * 8;
        const T* x1 = reinterpret_cast<const T*>(p.x) + (row0 + max(t1, 0)) * p.K + q * 8;
        constexpr int U = NT <= 2 ? 4 : NT <= 4 ? 2 : 1;     // chunks in flight
        for (int rb = 0; rb < rank; rb += NT * 8) {
            float acc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
            const T* ab = a + (int64_t)(rb + g) * K + q * 8;
            const int64_t a_step = (int64_t)8 * K;
            for (int c = c_lo + warp; c < c_hi; c += kWarps * U) {
                uint4 xa[U], xb[U], w[U][NT];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = (c + u * kWarps) * 32;
                    const bool in = c + u * kWarps < c_hi && k + q * 8 < K;
                    xa[u] = in && r0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
                    xb[u] = in && r1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        w[u][j] = in && rb + j * 8 + g < rank ? __ldg(reinterpret_cast<const uint4*>(ab + j * a_step + k)) : zero;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        mma16(acc[j], xa[u].x, xb[u].x, xa[u].y, xb[u].y, w[u][j].x, w[u][j].y, (const T*)nullptr);
                        mma16(acc[j], xa[u].z, xb[u].z, xa[u].w, xb[u].w, w[u][j].z, w[u][j].w, (const T*)nullptr);
                    }
            }
            const int width = min(NT * 8, rank8 - rb);       // of this block of ranks, in whole tiles
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (j * 8 >= width) break;
                float* dst = part + (warp * kRows + g) * width + j * 8 + 2 * q;
                if (r0) {
                    dst[0] = acc[j][0];
                    dst[1] = acc[j][1];
                }
                if (r1) {
                    dst[8 * width] = acc[j][2];
                    dst[8 * width + 1] = acc[j][3];
                }
            }
            __syncthreads();
            for (int r = warp; r < kRows; r += kWarps) {
                if (row_of[r] < 0) continue;
                for (int c = lane; c < width; c += 32) {
                    float s = 0.0f;
#pragma unroll
                    for (int v = 0; v < kWarps; ++v) s += part[(v * kRows + r) * width + c];
                    own[r * rank8 + rb + c] = s;
                }
            }
            __syncthreads();
        }
        // ---- the CTAs' sums meet in every CTA: a warp per row, as two terms and a power of two ----
        cluster_arrive();
        cluster_wait();
        for (int r = warp; r < kRows; r += kWarps) {
            const bool used = row_of[r] >= 0;
            float v[kMaxRank / 32], top = 0.0f;
#pragma unroll
            for (int i = 0; i < kMaxRank / 32; ++i) {
                v[i] = 0.0f;
                const int at_k = i * 32 + lane;
                if (i * 32 < rank && used)
                    for (int c0 = 0; c0 < (int)ctas; c0 += kGather) {
                        float u[kGather];
#pragma unroll
                        for (int c = 0; c < kGather; ++c) u[c] = c0 + c < (int)ctas && at_k < rank ? load_remote(own + r * rank8 + at_k, c0 + c) : 0.0f;
#pragma unroll
                        for (int c = 0; c < kGather; ++c) v[i] += u[c];
                    }
                top = fmaxf(top, fabsf(v[i]));
            }
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            // the largest value to [2^13, 2^14); the factor and its inverse are exact
            const int e = top > 0.0f && top < INFINITY ? min(126, 13 + 127 - (int)(__float_as_uint(top) >> 23)) : 0;
            const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int i = 0; i < kMaxRank / 32; ++i) {
                const int k = i * 32 + lane;
                if (k >= (rank16 + 31) / 32 * 32) continue;
                const float t = v[i] * up;
                const T h = from_f32<T>(t);
                const float rest = t - to_f32(h);
                hi[r * at.low_stride + k] = h;
                lo[r * at.low_stride + k] = from_f32<T>(fabsf(rest) < INFINITY ? rest : 0.0f);
            }
            if (lane == 0) row_scale[r] = down * (p.scaling && id >= 0 ? p.scaling[id] : 1.0f);
        }
        cluster_arrive();                                    // nobody reads this CTA's sums any more: waited for at the end
        __syncthreads();

        // ---- times B ----
        float f[2];
        f[0] = row_scale[g];
        f[1] = row_scale[g + 8];
        const int64_t at0 = (row0 + t0) * p.N + q * 8, at1 = (row0 + t1) * p.N + q * 8;
        for (int s = s_first; s < strips; s += s_step, b_lane += b_step) {
            const int n = s * 32 + q * 8;
            uint4 was[2] = {zero, zero};                     // y of the lane's columns
            if (y != nullptr)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if ((half ? t1 : t0) < 0 || n >= N) continue;
                    const T* src = y + (half ? at1 : at0) + s * 32;
                    if (vector_rows) {
                        was[half] = *reinterpret_cast<const uint4*>(src);
                    } else {
                        T e[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) e[i] = n + i < N ? src[i] : from_f32<T>(0.0f);
                        was[half] = *reinterpret_cast<const uint4*>(e);
                    }
                }
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
            int k0 = 0;
            do {
                Piece next[4];
                if constexpr (DEPTH > 0) {
                    if (k0 < rank) {
                        cp_async_wait<DEPTH - 1>();
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const Piece*>(ring + (ring_at * 4 + j) * 32);
                        const int k = k0 + q * kPer;
                        if (ragged && k < rank && k + kPer > rank)
#pragma unroll
                            for (int j = 0; j < 4; ++j) keep_ranks(w[j], rank - k);
                    }
                } else {
                    if (k0 + kStep < rank) load_b(next, b_lane, s, k0 + kStep);
                    else if (s + s_step < strips) load_b(next, b_lane + b_step, s + s_step, 0);
                }
                if (k0 < rank) {
                    const int k = k0 + q * kPer;
                    const Piece h0 = *reinterpret_cast<const Piece*>(hi + g * at.low_stride + k), h1 = *reinterpret_cast<const Piece*>(hi + (g + 8) * at.low_stride + k);
                    const Piece l0 = *reinterpret_cast<const Piece*>(lo + g * at.low_stride + k), l1 = *reinterpret_cast<const Piece*>(lo + (g + 8) * at.low_stride + k);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma16(acc[j], h0.x, h1.x, h0.y, h1.y, w[j].x, w[j].y, (const T*)nullptr);
                        mma16(acc[j], l0.x, l1.x, l0.y, l1.y, w[j].x, w[j].y, (const T*)nullptr);
                    }
                    if constexpr (kPer == 8) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            mma16(acc[j], h0.z, h1.z, h0.w, h1.w, w[j].z, w[j].w, (const T*)nullptr);
                            mma16(acc[j], l0.z, l1.z, l0.w, l1.w, w[j].z, w[j].w, (const T*)nullptr);
                        }
                    }
                }
                if constexpr (DEPTH > 0) {
                    if (k0 < rank) copy_round();             // behind the products: the slot has been read
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = next[j];
                }
                k0 += kStep;
            } while (k0 < rank);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if ((half ? t1 : t0) < 0 || n >= N) continue;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = acc[i >> 1][2 * half + (i & 1)] * f[half];
                if (y != nullptr) {
                    const T* e = reinterpret_cast<const T*>(&was[half]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = id < 0 ? to_f32(e[i]) : v[i] + to_f32(e[i]);
                }
                const int64_t to = (half ? at1 : at0) + s * 32;
                if (p.out32) {
                    float* dst = reinterpret_cast<float*>(p.out) + to;
                    if (vector_rows) {
                        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (n + i < N) dst[i] = v[i];
                    }
                } else {
                    T o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(v[i]);
                    T* dst = reinterpret_cast<T*>(p.out) + to;
                    if (vector_rows) {
                        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (n + i < N) dst[i] = o[i];
                    }
                }
            }
        }
        cluster_wait();                                      // also: no CTA overwrites its sums for the next row while another reads them
        __syncthreads();
    }
}

template <typename T> int cluster_form(const LoraParams& p, cudaStream_t stream) {
    const bool narrow = p.R <= 16 || p.R % 8 != 0 || ((uintptr_t)p.b & 15u) != 0, wide = !narrow && p.R > 32;
    const int64_t windows = (p.rows + kWindow - 1) / kWindow, slots = (int64_t)sm_count() * 2;
    // CTAs per cluster.  As many as leave every row a cluster of its own on the GPU at once; four at least (eight where a group reads a MB of
    // factors, and the rows fill no window, or 4 MB: few groups then) but fewer when the groups of 16 rows alone fill the GPU.  With
    // the projection, us for 4 / 8 / 16: one row, rank 16, 4096 x 4096: 12.2 / 11.0 / 10.7; 32 rows, rank 64, 6144 x 4096: 33.7 / 29.1 / 35.5; 128 rows of 32
    // adapters, rank 16, 4096 x 4096: 24.0 / 26.9 / 36.7; 512 rows, rank 64, 14336 x 4096: 113.3 / 121.0 / 133; 64 rows of 8 adapters of rank 64, 6144 x
    // 4096: 26.3 / 23.9, 512: 61.8 / 66.6; of rank 256, 512 rows: 104.5 / 96.9.
    int ctas = tuning_get("lora.cluster");
    if (ctas <= 0) {
        const int64_t factors = (int64_t)p.R * (p.K + p.N);      // values that a group reads
        const int least = factors >= 2048 * 1024 || (factors >= 512 * 1024 && p.rows < kWindow) ? 8 : 4;
        ctas = 16;
        while (ctas > least && p.rows * ctas > slots) ctas /= 2;
        while (ctas > 1 && (p.rows + kRows - 1) / kRows * ctas > slots) ctas /= 2;
    }
    // clusters per window: one for each of its rows, as far as the GPU holds them
    const int64_t rows = std::min<int64_t>(p.rows, kWindow), per_window = std::min(rows, std::max<int64_t>(1, slots / ctas / windows));
    const int64_t clusters = windows * per_window;
    // clusters per group at most, when there are more of them than groups: each warp keeps two rounds of B or more (with projections of 6144 x 4096:
    // 128 rows of one adapter of rank 64 34.3 -> 32.0 us, of eight adapters of rank 256 71.1 -> 59.0; one round: 32 rows of 8 adapters of rank 32 17.7 -> 18.8)
    const int64_t turns = ((p.N + 31) / 32 + ctas * 8 - 1) / (ctas * 8), rounds = turns * ((p.R + (narrow ? 15 : 31)) / (narrow ? 16 : 32));
    const int max_slices = (int)std::max<int64_t>(1, std::min(turns, rounds / 2));
    if (clusters > INT32_MAX / ctas) return B200Q_ERR_UNSUPPORTED;
    const int warps = 8;
    const size_t smem = lora_smem(p.R, warps, ring_depth(narrow ? 2 : 8)).bytes;
    const bool sliced = max_slices > 1 && 2 * ((rows + kRows - 1) / kRows) <= per_window;      // there can be clusters enough
    void (*kernel)(const LoraParams, int, int, int) =
        sliced ? (narrow ? lora_cluster_kernel<T, 2, 8, true> : wide ? lora_cluster_kernel<T, 8, 8, true> : lora_cluster_kernel<T, 4, 8, true>)
               : (narrow ? lora_cluster_kernel<T, 2, 8, false> : wide ? lora_cluster_kernel<T, 8, 8, false> : lora_cluster_kernel<T, 4, 8, false>);
    if (smem > 40 * 1024 &&      // with the static part beyond what needs no asking (one value for all calls: two threads may launch the same kernel)
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lora_smem(kMaxRank, warps, ring_depth(8)).bytes) != cudaSuccess)
        return B200Q_ERR_LAUNCH;
    if (ctas > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return B200Q_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * ctas));
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tuning_get("no_pdl") ? 1 : 2;
    const int vector_rows = p.N % 8 == 0 && (((uintptr_t)p.y | (uintptr_t)p.out) & 15u) == 0;      // results in 16-byte pieces
    return cudaLaunchKernelEx(&cfg, kernel, p, (int)per_window, max_slices, vector_rows) == cudaSuccess ? finish_launch() : B200Q_ERR_LAUNCH;
}
bool cluster_takes(const LoraParams& p) {
    return p.K % 8 == 0 && p.K < (1 << 30) && p.N < (1 << 30) && p.R % 4 == 0 && p.R <= kMaxRank && (((uintptr_t)p.x | (uintptr_t)p.a) & 15u) == 0 && ((uintptr_t)p.b & 7u) == 0;
}

}  // namespace

size_t lora_workspace_impl(int64_t rows, int R) { return rows <= 0 || R <= 0 ? 0 : 4 * (size_t)rows * (size_t)R; }

int lora_rows(const LoraParams& p, int dtype, size_t ws_bytes, cudaStream_t stream) {
    if (cluster_takes(p)) return dtype == B200Q_F16 ? cluster_form<__half>(p, stream) : cluster_form<__nv_bfloat16>(p, stream);
    if (p.low == nullptr || ws_bytes < lora_workspace_impl(p.rows, p.R)) return B200Q_ERR_WORKSPACE;
    return dtype == B200Q_F16 ? any_size<__half>(p, stream) : any_size<__nv_bfloat16>(p, stream);
}

int lora_add_impl(const void* x, const void* y, void* out, const void* a, const void* b, const float* scaling, const int32_t* ranks,
                  const int32_t* ids, int64_t rows, int64_t N, int64_t K, int L, int R, int dtype, void* ws, size_t ws_bytes,
                  cudaStream_t stream) {
    if (x == nullptr || out == nullptr || a == nullptr || b == nullptr || ids == nullptr) return B200Q_ERR_BAD_ARG;
    if (rows <= 0 || N <= 0 || K <= 0 || L <= 0 || R <= 0 || !is_act_dtype(dtype)) return B200Q_ERR_BAD_ARG;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < lora_workspace_impl(rows, R)) return B200Q_ERR_WORKSPACE;
    return lora_rows({x, y, out, a, b, scaling, ranks, ids, (float*)ws, rows, K, N, L, R, 0}, dtype, ws_bytes, stream);
}

// A few rows of small ranks: one launch of the integer matvec, in which every CTA forms A x itself, as long as that takes its 16 warps eight rounds
// of 1024 values or less.  Two launches -> one, us, rows / rank: 4096 x 4096 q4 1/16 10.9 -> 6.8, 1/32 11.0 -> 7.7, 2/16 12.6 -> 10.1, 4/8 14.0 -> 11.8;
// 2048 x 2048 4/16 11.8 -> 10.7; 14336 x 4096 1/16 17.4 -> 11.5.  Beyond: 4096 x 4096 2/32 12.7 -> 13.4, 4/16 14.0 -> 16.2; 4096 x 14336 1/8 16.8 -> 17.5.
constexpr int64_t kFusedRounds = 8;
// More: the adapters' rows in fp32, then the matvec that adds them before its one rounding.
static size_t low_rows_bytes(int64_t rows, int64_t N) { return (4 * (size_t)rows * (size_t)N + 255) / 256 * 256; }
size_t lora_qmatvec_workspace_impl(int64_t rows, int64_t N, int R) {
    return rows <= 0 || N <= 0 || R <= 0 ? 0 : low_rows_bytes(rows, N) + lora_workspace_impl(rows, R);
}
int lora_qmatvec_impl(int bits, const void* x, const uint8_t* codes, const void* scales, const void* zeros, const void* residual, void* y,
                      const void* a, const void* b, const float* scaling, const int32_t* ranks, const int32_t* ids, int rows, int64_t N, int64_t K,
                      int group_size, int L, int R, int act_dtype, int scale_dtype, void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (x == nullptr || codes == nullptr || scales == nullptr || y == nullptr || a == nullptr || b == nullptr || ids == nullptr) return B200Q_ERR_BAD_ARG;
    if ((bits != 4 && bits != 8) || rows <= 0 || N <= 0 || K <= 0 || L <= 0 || R <= 0 || group_size <= 0 || !is_act_dtype(act_dtype) ||
        !is_scale_dtype(scale_dtype))
        return B200Q_ERR_BAD_ARG;
    if (N > INT32_MAX || K > INT32_MAX) return B200Q_ERR_UNSUPPORTED;
    if (ws == nullptr || ((uintptr_t)ws & 15u) != 0 || ws_bytes < lora_qmatvec_workspace_impl(rows, N, R)) return B200Q_ERR_WORKSPACE;
    const int fused = tuning_get("lora.fused");
    if (fused >= 0 && rows <= 4 && (fused > 0 || (rows * (int64_t)R + 15) / 16 * ((K + 1023) / 1024) <= kFusedRounds)) {
        const int rc = lora_rows_qmatvec(bits, x, codes, scales, zeros, residual, y, rows, N, K, group_size, act_dtype, scale_dtype,
                                         {a, b, scaling, ranks, ids, L, R}, stream);
        if (rc != B200Q_ERR_UNSUPPORTED) return rc;
    }
    const size_t low = low_rows_bytes(rows, N);
    const int rc = lora_rows({x, residual, ws, a, b, scaling, ranks, ids, (float*)((uint8_t*)ws + low), rows, K, N, L, R, 1}, act_dtype, ws_bytes - low, stream);
    if (rc != B200Q_OK) return rc;
    return qmatvec_impl(bits, x, codes, scales, zeros, nullptr, y, rows, N, K, group_size, act_dtype, scale_dtype, nullptr, nullptr, B200Q_F16, 0.0f,
                        nullptr, nullptr, stream, (const float*)ws);
}

}  // namespace b200q
