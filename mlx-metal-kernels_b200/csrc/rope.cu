// Rotary positions on the heads of queries and keys, with an optional RMSNorm per head in front, into tensors or into the
// paged key/value cache.
//
//   y = x                                    or, with a weight w [D]:  y = x * rsqrt(mean(x^2) + eps) * w
//   (u, v) -> (u cos - v sin, u sin + v cos) for the pairs of the first R dimensions of the head:
//       interleaved: u = y[2i], v = y[2i + 1]        half: u = y[i], v = y[i + R/2]           i < R/2
//   with cos / sin [table_len, R/2] in fp32 at the token's position; the other D - R dimensions pass through.
//   Everything is fp32 and rounded once, to the type of the rows.
//
// The append form takes the fused rows [q heads | k heads | v heads] of a projection, returns the q heads and writes the k heads
// (normalised, rotated) and the v heads (as they are) to slot pos % P of page block_table[sequence, pos / P]: as they are, or
// quantised from the rounded values with the cache's rule (see stack.cu).
//
#include "common.cuh"

#include <algorithm>

namespace b200q {

B200Q_DEFINE_STATUS_WORD(rope_read_status)

namespace {

enum HeadKind : int { KIND_Q = 0, KIND_K = 1, KIND_V = 2 };
enum CacheKind : int { NO_CACHE = 0, CACHE_Q4 = 4, CACHE_Q8 = 8, CACHE_PLAIN = 16 };

struct RopeParams {
    const void* in[3];            // q, k, v heads; element strides below
    void* out[3];                 // q_out and, without a cache, k_out
    int64_t in_token[3], in_head[3], out_token[3], out_head[3];
    const void* weight[3];        // per-head norm weights [D] or null (never for v)
    const float* cos_table;
    const float* sin_table;
    const int32_t* positions;     // [T]
    const int32_t* sequences;     // [T] or null: token t belongs to sequence t; negative: padding
    const int32_t* block_table;   // [B, max_blocks]
    void* codes[3];               // k and v pages at KIND_K, KIND_V
    __half* scales[3];
    int64_t T, table_len, num_pages;
    int heads[3];                 // heads per kind
    int B, max_blocks, P, D, R, G, w_dtype;
    float eps;
};

// (u, v) turned: separately rounded products and one sum, as elementwise operations give it
__device__ __forceinline__ float turn_u(float u, float v, float c, float s) { return __fsub_rn(__fmul_rn(u, c), __fmul_rn(v, s)); }
__device__ __forceinline__ float turn_v(float u, float v, float c, float s) { return __fadd_rn(__fmul_rn(u, s), __fmul_rn(v, c)); }

// Page slot of a token, or -1: nothing is written.  Padding (a negative sequence) is no event; a sequence or a position
// without a page is.
__device__ __forceinline__ int64_t cache_row(const RopeParams& p, int64_t t, int pos, int seq, bool report) {
    if (seq < 0) return -1;
    int page = -1;
    if (seq < p.B && pos >= 0 && pos / p.P < p.max_blocks) page = p.block_table[(size_t)seq * p.max_blocks + pos / p.P];
    if (page < 0 || page >= p.num_pages) {
        if (report) atomicMax(&g_device_status, (int)EV_KV_PAGE_UNASSIGNED);
        return -1;
    }
    return (int64_t)page * p.P + pos % p.P;
}

template <int CACHE> __device__ __forceinline__ uint32_t kv_code(float v, float scale) {
    constexpr float limit = CACHE == CACHE_Q8 ? 127.0f : 7.0f, offset = CACHE == CACHE_Q8 ? 128.0f : 8.0f;
    return (uint32_t)(int)(fminf(fmaxf(rintf(__fdiv_rn(v, scale)), -limit), limit) + offset);
}

// Any head size, rotary size, group size, stride and alignment: one warp per (token, head), the head in shared memory.
constexpr int kAnyWarps = 4, kAnyMaxDim = 1024;
template <typename T, int CACHE>
__global__ void __launch_bounds__(kAnyWarps * 32) rope_any_kernel(const __grid_constant__ RopeParams p, bool half_layout, int64_t units) {
    extern __shared__ float smem[];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, D = p.D, half = p.R / 2;
    float* y = smem + (threadIdx.x >> 5) * (size_t)D;
    const int64_t unit = (int64_t)blockIdx.x * kAnyWarps + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int per_token = p.heads[0] + p.heads[1] + p.heads[2];
    const int64_t t = unit / per_token;
    int h = (int)(unit - t * per_token), kind = KIND_Q;
    if (h >= p.heads[0]) { h -= p.heads[0]; kind = KIND_K; }
    if (kind == KIND_K && h >= p.heads[1]) { h -= p.heads[1]; kind = KIND_V; }
    const int pos = p.positions[t];
    const int seq = CACHE != NO_CACHE ? (p.sequences ? p.sequences[t] : (int)t) : 0;
    const bool padding = CACHE != NO_CACHE && seq < 0, in_table = pos >= 0 && pos < p.table_len;
    if (kind != KIND_V && !in_table && !padding && lane == 0) atomicMax(&g_device_status, (int)EV_ROPE_POSITION);
    const T* src = reinterpret_cast<const T*>(p.in[kind]) + t * p.in_token[kind] + (int64_t)h * p.in_head[kind];
    float ss = 0.0f;
    for (int d = lane; d < D; d += 32) {
        const float v = to_f32(src[d]);
        y[d] = v;
        ss = fmaf(v, v, ss);
    }
    if (p.weight[kind] != nullptr) {
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float inv = rsqrtf(ss / (float)D + p.eps);
        for (int d = lane; d < D; d += 32) y[d] = y[d] * inv * load_as_f32(p.weight[kind], p.w_dtype, d);
    }
    __syncwarp();
    if (kind != KIND_V && in_table && !padding) {
        for (int i = lane; i < half; i += 32) {
            const float c = p.cos_table[(int64_t)pos * half + i], s = p.sin_table[(int64_t)pos * half + i];
            const int iu = half_layout ? i : 2 * i, iv = half_layout ? i + half : 2 * i + 1;
            const float u = y[iu], v = y[iv];
            y[iu] = turn_u(u, v, c, s);
            y[iv] = turn_v(u, v, c, s);
        }
        __syncwarp();
    }
    if (CACHE == NO_CACHE || kind == KIND_Q) {
        T* dst = reinterpret_cast<T*>(p.out[kind]) + t * p.out_token[kind] + (int64_t)h * p.out_head[kind];
        for (int d = lane; d < D; d += 32) dst[d] = from_f32<T>(padding ? 0.0f : y[d]);
        return;
    }
    const int64_t row_index = cache_row(p, t, pos, seq, lane == 0);
    if (row_index < 0) return;
    const int64_t row = row_index * p.heads[kind] + h;
    if (CACHE == CACHE_PLAIN) {
        for (int d = lane; d < D; d += 32) reinterpret_cast<T*>(p.codes[kind])[row * D + d] = from_f32<T>(y[d]);
        return;
    }
    // lanes take bytes of codes: two values each in q4, whose groups may differ
    const int groups = (D + p.G - 1) / p.G, per_byte = CACHE == CACHE_Q4 ? 2 : 1, bytes = (D + per_byte - 1) / per_byte;
    for (int d = lane; d < D; d += 32) y[d] = to_f32(from_f32<T>(y[d]));
    __syncwarp();
    constexpr float limit = CACHE == CACHE_Q8 ? 127.0f : 7.0f;
    auto scale_of = [&](int g) {
        float m = 0.0f;
        for (int d = g * p.G; d < min(D, (g + 1) * p.G); ++d) m = fmaxf(m, fabsf(y[d]));
        return __fdiv_rn(fmaxf(m, 1e-8f), limit);
    };
    for (int g = lane; g < groups; g += 32) p.scales[kind][row * groups + g] = __float2half_rn(scale_of(g));
    for (int i = lane; i < bytes; i += 32) {
        uint32_t byte = 0;
        for (int k = 0; k < per_byte; ++k) {
            const int d = i * per_byte + k;
            if (d < D) byte |= kv_code<CACHE>(y[d], scale_of(d / p.G)) << (4 * k);
        }
        reinterpret_cast<uint8_t*>(p.codes[kind])[row * bytes + i] = (uint8_t)byte;
    }
}

template <typename K, typename... A>
int launch(K kernel, int64_t blocks, int threads, size_t smem, cudaStream_t stream, A... args) {
    if (blocks > INT32_MAX) return B200Q_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tuning_get("no_pdl") ? 0 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) return B200Q_ERR_LAUNCH;
    return finish_launch();
}

template <typename T, int CACHE>
int dispatch(RopeParams& p, bool half_layout, cudaStream_t stream) {
    const int64_t units = p.T * (p.heads[0] + p.heads[1] + p.heads[2]);
    return launch(rope_any_kernel<T, CACHE>, (units + kAnyWarps - 1) / kAnyWarps, kAnyWarps * 32, sizeof(float) * kAnyWarps * p.D, stream, p,
                  half_layout, units);
}

}  // namespace

int head_rope_impl(const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, const void* q_weight,
                   const void* k_weight, int w_dtype, float eps, const float* cos_table, const float* sin_table,
                   const int32_t* positions, int64_t table_len, int rotary_dim, int half_layout, int64_t T, int Hq, int Hkv, int D,
                   int dtype, cudaStream_t stream) {
    if (q == nullptr || q_out == nullptr || strides == nullptr || cos_table == nullptr || sin_table == nullptr || positions == nullptr ||
        (Hkv > 0 && (k == nullptr || k_out == nullptr)))
        return B200Q_ERR_BAD_ARG;
    if (T <= 0 || Hq <= 0 || Hkv < 0 || D <= 0 || table_len <= 0 || rotary_dim <= 0 || rotary_dim > D || rotary_dim % 2 != 0 ||
        !is_act_dtype(dtype) || ((q_weight || k_weight) && !is_scale_dtype(w_dtype)))
        return B200Q_ERR_BAD_ARG;
    if (D > kAnyMaxDim) return B200Q_ERR_UNSUPPORTED;
    RopeParams p = {};
    p.in[KIND_Q] = q; p.out[KIND_Q] = q_out;
    p.in_token[KIND_Q] = strides[0]; p.in_head[KIND_Q] = strides[1]; p.out_token[KIND_Q] = strides[2]; p.out_head[KIND_Q] = strides[3];
    if (Hkv > 0) {
        p.in[KIND_K] = k; p.out[KIND_K] = k_out;
        p.in_token[KIND_K] = strides[4]; p.in_head[KIND_K] = strides[5]; p.out_token[KIND_K] = strides[6]; p.out_head[KIND_K] = strides[7];
    }
    p.weight[KIND_Q] = q_weight; p.weight[KIND_K] = k_weight;
    p.cos_table = cos_table; p.sin_table = sin_table; p.positions = positions;
    p.T = T; p.table_len = table_len; p.heads[KIND_Q] = Hq; p.heads[KIND_K] = Hkv;
    p.P = 1; p.D = D; p.R = rotary_dim; p.G = 8; p.w_dtype = w_dtype; p.eps = eps;
    return dtype == B200Q_F16 ? dispatch<__half, NO_CACHE>(p, half_layout != 0, stream)
                              : dispatch<__nv_bfloat16, NO_CACHE>(p, half_layout != 0, stream);
}

int norm_rope_kv_append_impl(const void* qkv, int64_t qkv_stride, const float* cos_table, const float* sin_table, int64_t table_len,
                             int rotary_dim, int half_layout, const int32_t* positions, const int32_t* sequences,
                             const int32_t* block_table, int B, int max_blocks, const void* q_weight, const void* k_weight, int w_dtype,
                             float eps, void* q_out, int kv_bits, void* k_pages, void* v_pages, void* k_scales, void* v_scales, int64_t T,
                             int Hq, int Hkv, int D, int page_size, int64_t num_pages, int group_size, int dtype, cudaStream_t stream) {
    if (qkv == nullptr || cos_table == nullptr || sin_table == nullptr || positions == nullptr || block_table == nullptr ||
        q_out == nullptr || k_pages == nullptr || v_pages == nullptr)
        return B200Q_ERR_BAD_ARG;
    if (kv_bits != 4 && kv_bits != 8 && kv_bits != 16) return B200Q_ERR_BAD_ARG;
    if (kv_bits != 16 && (k_scales == nullptr || v_scales == nullptr || group_size <= 0)) return B200Q_ERR_BAD_ARG;
    if (T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || table_len <= 0 || rotary_dim <= 0 || rotary_dim > D || rotary_dim % 2 != 0 || B <= 0 ||
        max_blocks <= 0 || page_size <= 0 || num_pages <= 0 || !is_act_dtype(dtype) || qkv_stride < (int64_t)(Hq + 2 * (int64_t)Hkv) * D ||
        ((q_weight || k_weight) && !is_scale_dtype(w_dtype)) || (sequences == nullptr && T > B))
        return B200Q_ERR_BAD_ARG;
    if (D > kAnyMaxDim) return B200Q_ERR_UNSUPPORTED;
    RopeParams p = {};
    const int64_t heads[3] = {Hq, Hkv, Hkv}, first[3] = {0, Hq, (int64_t)Hq + Hkv};
    for (int i = 0; i < 3; ++i) {
        p.in[i] = reinterpret_cast<const uint16_t*>(qkv) + first[i] * D;
        p.in_token[i] = qkv_stride;
        p.in_head[i] = D;
        p.heads[i] = (int)heads[i];
    }
    p.out[KIND_Q] = q_out; p.out_token[KIND_Q] = (int64_t)Hq * D; p.out_head[KIND_Q] = D;
    p.weight[KIND_Q] = q_weight; p.weight[KIND_K] = k_weight;
    p.cos_table = cos_table; p.sin_table = sin_table; p.positions = positions; p.sequences = sequences; p.block_table = block_table;
    p.codes[KIND_K] = k_pages; p.codes[KIND_V] = v_pages;
    p.scales[KIND_K] = (__half*)k_scales; p.scales[KIND_V] = (__half*)v_scales;
    p.T = T; p.table_len = table_len; p.num_pages = num_pages; p.B = B; p.max_blocks = max_blocks; p.P = page_size;
    p.D = D; p.R = rotary_dim; p.G = kv_bits == 16 ? 8 : group_size; p.w_dtype = w_dtype; p.eps = eps;
    const bool half = half_layout != 0;
    if (dtype == B200Q_F16) {
        if (kv_bits == 16) return dispatch<__half, CACHE_PLAIN>(p, half, stream);
        return kv_bits == 8 ? dispatch<__half, CACHE_Q8>(p, half, stream) : dispatch<__half, CACHE_Q4>(p, half, stream);
    }
    if (kv_bits == 16) return dispatch<__nv_bfloat16, CACHE_PLAIN>(p, half, stream);
    return kv_bits == 8 ? dispatch<__nv_bfloat16, CACHE_Q8>(p, half, stream) : dispatch<__nv_bfloat16, CACHE_Q4>(p, half, stream);
}

}  // namespace b200q
