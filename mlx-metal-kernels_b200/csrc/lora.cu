// Low-rank adapters of many requests beside one shared projection.
//
//   out[t] = cast(y[t] + s[l] * B[l] (A[l] x[t])),   l = ids[t];   ids[t] < 0: out[t] = y[t]
//
// A [L, R, K] and B [L, N, R] hold the factors of L adapters, of which adapter l uses the first ranks[l] of R; x [rows, K], y and out
// [rows, N] (out may be y).  Products are summed in fp32, the R values between the factors stay in fp32 (or in as many bits), and the
// sum with y is rounded once.
#include "common.cuh"

#include <algorithm>

namespace b200q {

B200Q_DEFINE_STATUS_WORD(lora_read_status)

namespace {

struct LoraParams {
    const void* x;            // [rows, K]
    const void* y;            // [rows, N]
    void* out;                // [rows, N]
    const void* a;            // [L, R, K]
    const void* b;            // [L, N, R]
    const float* scaling;     // [L] or null: 1
    const int32_t* ranks;     // [L] or null: R
    const int32_t* ids;       // [rows]
    float* low;               // [rows, R] scratch of the general kernels
    int64_t rows, K, N;
    int L, R;
};

// Adapter of a row, or -1.
__device__ __forceinline__ int adapter_of(const LoraParams& p, int64_t row) {
    const int id = p.ids[row];
    return id < p.L ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraParams& p, int id) { return p.ranks ? max(0, min(p.R, p.ranks[id])) : p.R; }

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
        const float y = to_f32(reinterpret_cast<const T*>(p.y)[it]);
        float s = 0.0f;
        if (id >= 0) {
            const T* b = reinterpret_cast<const T*>(p.b) + ((int64_t)id * p.N + n) * p.R;
            const float* low = p.low + row * p.R;
            const int rank = rank_of(p, id);
            for (int r = 0; r < rank; ++r) s = fmaf(to_f32(b[r]), low[r], s);
            if (p.scaling) s *= p.scaling[id];
        }
        reinterpret_cast<T*>(p.out)[it] = id < 0 ? reinterpret_cast<const T*>(p.y)[it] : from_f32<T>(y + s);
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

}  // namespace

size_t lora_workspace_impl(int64_t rows, int R) { return rows <= 0 || R <= 0 ? 0 : 4 * (size_t)rows * (size_t)R; }

int lora_add_impl(const void* x, const void* y, void* out, const void* a, const void* b, const float* scaling, const int32_t* ranks,
                  const int32_t* ids, int64_t rows, int64_t N, int64_t K, int L, int R, int dtype, void* ws, size_t ws_bytes,
                  cudaStream_t stream) {
    if (x == nullptr || y == nullptr || out == nullptr || a == nullptr || b == nullptr || ids == nullptr) return B200Q_ERR_BAD_ARG;
    if (rows <= 0 || N <= 0 || K <= 0 || L <= 0 || R <= 0 || !is_act_dtype(dtype)) return B200Q_ERR_BAD_ARG;
    if (ws == nullptr || ws_bytes < lora_workspace_impl(rows, R)) return B200Q_ERR_WORKSPACE;
    const LoraParams p = {x, y, out, a, b, scaling, ranks, ids, (float*)ws, rows, K, N, L, R};
    return dtype == B200Q_F16 ? any_size<__half>(p, stream) : any_size<__nv_bfloat16>(p, stream);
}

}  // namespace b200q
