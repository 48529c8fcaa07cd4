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
// quantised from the rounded values: scale = max(max|v|, 1e-8) * (1/127 | 1/7), code = clip(rint(v / scale)) + (128 | 8).
//
// Bound by HBM for prompts and by latency for a few tokens.  A head is taken by D/16 lanes, so that a lane has two 16-byte pieces
// of it: pieces l and l + D/16, which are the two halves of eight pairs in the half layout over whole heads.  One head per
// lane while all fit the GPU at once; else two (RUN) of one token, which share the token's cos / sin and the norm's weights, with four blocks
// per SM: the append of 8185 tokens of 48 heads with norms takes 48 us so, 56 with four heads and 68 with one.  From eight tokens per SM on rows
// come through a ring in shared memory: 44 us for them, 4.7 TB/s; 8192 tokens without norms 29 us, 5.8 TB/s.
#include "common.cuh"

#include <algorithm>

namespace b200q {

B200Q_DEFINE_STATUS_WORD(rope_read_status)

namespace {

constexpr int kThreads = 256;

enum HeadKind : int { KIND_Q = 0, KIND_K = 1, KIND_V = 2 };
enum Layout : int { INTERLEAVED = 0, HALF_WHOLE = 1, HALF_PART = 2 };
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
    int heads[3], runs[3];        // heads per kind, and groups of RUN of them
    int B, max_blocks, P, D, R, G, w_dtype;
    float eps;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8], const __half*) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    return *reinterpret_cast<const uint4*>(e);
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load_weight8(const void* w, int dtype, int i, float (&v)[8]) {
    if (dtype == B200Q_F32) {
        load8(reinterpret_cast<const float*>(w) + i, v);
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(w) + i));
        if (dtype == B200Q_F16) unpack8(u, v, (const __half*)nullptr);
        else unpack8(u, v, (const __nv_bfloat16*)nullptr);
    }
}

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

// two fp32 values in one 64-bit register, for the packed instructions
struct f32x2 { unsigned long long v; };
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(f32x2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

template <typename T> __device__ __forceinline__ void halves(uint32_t w, float& lo, float& hi);
template <> __device__ __forceinline__ void halves<__half>(uint32_t w, float& lo, float& hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
}
template <> __device__ __forceinline__ void halves<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
}
template <typename T> __device__ __forceinline__ uint32_t word(float lo, float hi);
template <> __device__ __forceinline__ uint32_t word<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t word<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The 16 values of a lane's two pieces as the u and the v of eight pairs: interleaved, each piece has four pairs; else piece 0 is
// the u and piece 1 the v.
struct Pairs { f32x2 u[4], v[4]; };
template <typename T, bool INTERLEAVE> __device__ __forceinline__ Pairs unpack(const uint4& p0, const uint4& p1) {
    const uint32_t w[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) halves<T>(w[i], lo[i], hi[i]);
    Pairs r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.u[i] = INTERLEAVE ? pair(lo[2 * i], lo[2 * i + 1]) : pair(lo[i], hi[i]);
        r.v[i] = INTERLEAVE ? pair(hi[2 * i], hi[2 * i + 1]) : pair(lo[4 + i], hi[4 + i]);
    }
    return r;
}
template <typename T, bool INTERLEAVE> __device__ __forceinline__ void pack(const Pairs& r, uint4& p0, uint4& p1) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float u0, u1, v0, v1;
        split(r.u[i], u0, u1);
        split(r.v[i], v0, v1);
        w[INTERLEAVE ? 2 * i : i] = INTERLEAVE ? word<T>(u0, v0) : word<T>(u0, u1);
        w[INTERLEAVE ? 2 * i + 1 : 4 + i] = INTERLEAVE ? word<T>(u1, v1) : word<T>(v0, v1);
    }
    p0 = make_uint4(w[0], w[1], w[2], w[3]);
    p1 = make_uint4(w[4], w[5], w[6], w[7]);
}
// Largest magnitude of a piece's eight values; NaN when one is.
template <typename T> __device__ __forceinline__ float piece_top(const uint4& u);
template <> __device__ __forceinline__ float piece_top<__half>(const uint4& u) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
template <> __device__ __forceinline__ float piece_top<__nv_bfloat16>(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
// The piece as the cache's rule sees it: its values and their largest magnitude, NaN passed over; `plain`: all are finite.
template <typename T> __device__ __forceinline__ float piece_values(const uint4& u, float (&v)[8], bool& plain) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) halves<T>(w[i], v[2 * i], v[2 * i + 1]);
    float top = piece_top<T>(u);
    plain = top < 3e38f;
    if (!plain) {
        top = 0.0f;
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    }
    return top;
}
// Scale of a group: max(top, 1e-8) times the rounded reciprocal of 127 or 7 - one instruction, and within a step of the quotient that the
// page quantiser (stack.cu) takes.  The codes are the same but for values exactly half way between two (14 v an odd multiple of the maximum in
// 4 bits), which may take the other one.
template <int CACHE> __device__ __forceinline__ float group_scale(float top) {
    return fmaxf(top, 1e-8f) * (1.0f / (CACHE == CACHE_Q8 ? 127.0f : 7.0f));
}
// Its codes.  rint(v / scale) with the quotient rounded as a division rounds it: the product with the correctly rounded reciprocal,
// corrected once by its exact remainder, is the correctly rounded quotient (Markstein's theorem) wherever it is large enough to matter.
template <int CACHE> __device__ __forceinline__ void store_codes(const float (&v)[8], float scale, bool plain, uint8_t* codes) {
    constexpr float limit = CACHE == CACHE_Q8 ? 127.0f : 7.0f, offset = CACHE == CACHE_Q8 ? 128.0f : 8.0f;
    constexpr float magic = 12582912.0f + offset;            // 1.5 2^23: adding it rounds to nearest even and leaves the code in the low byte
    constexpr uint32_t lowest = (uint32_t)(offset - limit), zero = (uint32_t)offset;
    const float inv = __frcp_rn(scale);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = v[i] * inv;
        c[i] = __float_as_uint(fmaf(fmaf(-q, scale, v[i]), inv, q) + magic);
    }
    if (!plain || !(scale < INFINITY)) {                     // as the rule has it: NaN becomes the lowest code, and beside an infinity all is zero
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(scale < INFINITY) || !(v[i] == v[i])) c[i] = fabsf(v[i]) < INFINITY ? zero : lowest;
    }
    auto bytes = [](uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) { return prmt(prmt(c0, c1, 0x0040u), prmt(c2, c3, 0x0040u), 0x5410u); };
    if (CACHE == CACHE_Q8) *reinterpret_cast<uint2*>(codes) = make_uint2(bytes(c[0], c[1], c[2], c[3]), bytes(c[4], c[5], c[6], c[7]));
    else *reinterpret_cast<uint32_t*>(codes) = bytes(c[0], c[2], c[4], c[6]) | bytes(c[1], c[3], c[5], c[7]) << 4;
}

// D a power of two from 32 to 256, R a multiple of 16, groups of whole pieces, everything aligned to 16 bytes.
template <typename T, int LAYOUT, int CACHE, int RUN>
__global__ void __launch_bounds__(kThreads, RUN == 1 ? 1 : LAYOUT == HALF_PART ? 3 : 4) rope_heads_kernel(const __grid_constant__ RopeParams p, int log_lanes, uint32_t units) {
    pdl_launch_dependents();
    pdl_wait();
    const int lanes = 1 << log_lanes;                        // lanes of a head: D / 16
    const int l = threadIdx.x & (lanes - 1);
    const uint32_t unit = blockIdx.x * (kThreads >> log_lanes) + (threadIdx.x >> log_lanes);
    const bool live = unit < units;
    const uint32_t per_token = p.runs[0] + p.runs[1] + p.runs[2], token = live ? unit / per_token : 0;
    const int64_t t = token;
    int run = live ? (int)(unit - token * per_token) : 0;
    int kind = KIND_Q;
    if (run >= p.runs[0]) { run -= p.runs[0]; kind = KIND_K; }
    if (kind == KIND_K && run >= p.runs[1]) { run -= p.runs[1]; kind = KIND_V; }
    const int h0 = run * RUN;
    const int count = live ? min(RUN, p.heads[kind] - h0) : 0;
    const int d0 = l * 8, d1 = (l + lanes) * 8;              // first dimension of the lane's two pieces

    const T* src = reinterpret_cast<const T*>(p.in[kind]) + t * p.in_token[kind] + (int64_t)h0 * p.in_head[kind];
    uint4 x0[RUN], x1[RUN], o0[RUN], o1[RUN];            // o: the partners of the pieces, where another lane owns them
    const int half = p.R / 2;
    const bool turns = kind != KIND_V;
    const int partner0 = d0 < half ? d0 + half : d0 - half, partner1 = d1 < half ? d1 + half : d1 - half;
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        x0[j] = x1[j] = o0[j] = o1[j] = make_uint4(0u, 0u, 0u, 0u);
        if (j < count) {
            const T* row = src + j * p.in_head[kind];
            x0[j] = *reinterpret_cast<const uint4*>(row + d0);
            x1[j] = *reinterpret_cast<const uint4*>(row + d1);
            if (LAYOUT == HALF_PART && turns) {
                if (d0 < p.R) o0[j] = *reinterpret_cast<const uint4*>(row + partner0);
                if (d1 < p.R) o1[j] = *reinterpret_cast<const uint4*>(row + partner1);
            }
        }
    }
    const int pos = live ? p.positions[t] : 0;
    const int seq = CACHE != NO_CACHE && live ? (p.sequences ? p.sequences[t] : (int)t) : 0;
    const float inv_d = 1.0f / (float)p.D;
    const bool padding = CACHE != NO_CACHE && seq < 0;
    const bool in_table = pos >= 0 && pos < p.table_len;
    const bool rotate = turns && in_table && !padding && live;
    if (live && turns && !in_table && !padding && l == 0) atomicMax(&g_device_status, (int)EV_ROPE_POSITION);

    // cos / sin: LAYOUT INTERLEAVED: four pairs of each piece; HALF_WHOLE: eight pairs; HALF_PART: eight pairs of each piece
    float c0[8], s0[8], c1[8], s1[8];
    if (rotate) {
        const float* ct = p.cos_table + (int64_t)pos * half;
        const float* st = p.sin_table + (int64_t)pos * half;
        if (LAYOUT == HALF_WHOLE) {
            load8(ct + d0, c0);
            load8(st + d0, s0);
        } else if (LAYOUT == HALF_PART) {
            if (d0 < p.R) { load8(ct + min(d0, partner0), c0); load8(st + min(d0, partner0), s0); }
            if (d1 < p.R) { load8(ct + min(d1, partner1), c1); load8(st + min(d1, partner1), s1); }
        } else {
            auto load4 = [](const float* q, float (&v)[8]) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(q));
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            };
            if (d0 < p.R) { load4(ct + d0 / 2, c0); load4(st + d0 / 2, s0); }
            if (d1 < p.R) { load4(ct + d1 / 2, c1); load4(st + d1 / 2, s1); }
        }
    }
    const void* weight = p.weight[kind];
    float w0[8], w1[8], wo0[8], wo1[8];
    if (weight != nullptr && live) {
        load_weight8(weight, p.w_dtype, d0, w0);
        load_weight8(weight, p.w_dtype, d1, w1);
        if (LAYOUT == HALF_PART) {
            if (d0 < p.R) load_weight8(weight, p.w_dtype, partner0, wo0);
            if (d1 < p.R) load_weight8(weight, p.w_dtype, partner1, wo1);
        }
    }
    int64_t row_index = -1;                                  // slot in the pool, in tokens
    if (CACHE != NO_CACHE && live && kind != KIND_Q) row_index = cache_row(p, t, pos, seq, l == 0);
    if (LAYOUT == HALF_PART) __syncwarp();                   // in place: nobody stores before the partners are loaded

#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        float a[8], b[8];
        unpack8(x0[j], a, (const T*)nullptr);
        unpack8(x1[j], b, (const T*)nullptr);
        float inv = 1.0f;
        if (weight != nullptr) {                             // uniform over the lanes of a head
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
            const unsigned group = (lanes == 32 ? 0xFFFFFFFFu : ((1u << lanes) - 1u)) << (threadIdx.x & 31 & ~(lanes - 1));
            for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor_sync(group, ss, o);
            inv = rsqrtf(ss / (float)p.D + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] = a[i] * inv * w0[i];
                b[i] = b[i] * inv * w1[i];
            }
        }
        if (rotate) {
            if (LAYOUT == HALF_WHOLE) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = a[i], v = b[i];
                    a[i] = turn_u(u, v, c0[i], s0[i]);
                    b[i] = turn_v(u, v, c0[i], s0[i]);
                }
            } else if (LAYOUT == HALF_PART) {
                auto half_part = [&](float (&x)[8], const uint4& other, const float (&wo)[8], const float (&c)[8], const float (&s)[8], bool low) {
                    float y[8];
                    unpack8(other, y, (const T*)nullptr);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (weight != nullptr) y[i] = y[i] * inv * wo[i];
                        x[i] = low ? turn_u(x[i], y[i], c[i], s[i]) : turn_v(y[i], x[i], c[i], s[i]);
                    }
                };
                if (d0 < p.R) half_part(a, o0[j], wo0, c0, s0, d0 < half);
                if (d1 < p.R) half_part(b, o1[j], wo1, c1, s1, d1 < half);
            } else {
                auto pairs = [](float (&x)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float u = x[2 * i], v = x[2 * i + 1];
                        x[2 * i] = turn_u(u, v, c[i], s[i]);
                        x[2 * i + 1] = turn_v(u, v, c[i], s[i]);
                    }
                };
                if (d0 < p.R) pairs(a, c0, s0);
                if (d1 < p.R) pairs(b, c1, s1);
            }
        }
        const uint4 y0 = pack8<T>(a), y1 = pack8<T>(b);
        if (CACHE == NO_CACHE || kind == KIND_Q) {
            if (j < count) {
                T* row = reinterpret_cast<T*>(p.out[kind]) + t * p.out_token[kind] + (int64_t)(h0 + j) * p.out_head[kind];
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4*>(row + d0) = padding ? zero : y0;
                *reinterpret_cast<uint4*>(row + d1) = padding ? zero : y1;
            }
        } else if (CACHE == CACHE_PLAIN) {
            if (j < count && row_index >= 0) {
                T* row = reinterpret_cast<T*>(p.codes[kind]) + (row_index * p.heads[kind] + h0 + j) * p.D;
                *reinterpret_cast<uint4*>(row + d0) = y0;
                *reinterpret_cast<uint4*>(row + d1) = y1;
            }
        } else {
            // the values as the cache sees them: rounded to T.  Group maxima over the G/8 neighbouring lanes; a group of the
            // whole head takes both pieces of every lane
            bool plain0, plain1;
            float m0 = piece_values<T>(y0, a, plain0), m1 = piece_values<T>(y1, b, plain1);
            const int pieces = p.G / 8;
            if (pieces > lanes) m0 = m1 = fmaxf(m0, m1);
            const unsigned group = (lanes == 32 ? 0xFFFFFFFFu : ((1u << lanes) - 1u)) << (threadIdx.x & 31 & ~(lanes - 1));
            for (int o = 1; o < min(pieces, lanes); o <<= 1) {
                m0 = fmaxf(m0, __shfl_xor_sync(group, m0, o));
                m1 = fmaxf(m1, __shfl_xor_sync(group, m1, o));
            }
            if (j < count && row_index >= 0) {
                const float q0 = group_scale<CACHE>(m0), q1 = group_scale<CACHE>(m1);
                const int64_t row = row_index * p.heads[kind] + h0 + j;
                auto store = [&](const float (&v)[8], float scale, bool plain, int d) {
                    store_codes<CACHE>(v, scale, plain, reinterpret_cast<uint8_t*>(p.codes[kind]) + (row * p.D + d) / (CACHE == CACHE_Q4 ? 2 : 1));
                    if (d % p.G == 0) p.scales[kind][row * (p.D / p.G) + d / p.G] = __float2half_rn(scale);
                };
                store(a, q0, plain0, d0);
                store(b, q1, plain1, d1);
            }
        }
    }
}

// ---- many tokens: rows through a ring in shared memory ---------------------------------------------------------------------
// The kernel above has no more bytes in flight than its registers hold.  Here a producer warp copies whole token rows (and their cos / sin
// rows) into a ring by bulk copies and finds the tokens' slots; consumer threads keep their heads and walk over the tokens.  A lane's two
// pieces are chosen so that it owns both halves of its pairs; its 16 values are held as two vectors (the u and the v of eight pairs), two
// values per 64-bit register, for the packed fp32 instructions.  Copying alone in this form takes 29.0 us for 8192 tokens of 40 heads, 36.5 for
// the append of 8185 tokens of 48; with norms the instructions bound it (51 % of issue slots): 44.  Three blocks per SM, with fewer registers: 62.
constexpr int kRingThreads = 384, kMaxStages = 12;
constexpr uint32_t kRingWaitLimit = 1u << 22;
constexpr uint32_t kRingBytes = 96 * 1024;      // of a block's stages: two blocks per SM
constexpr int kRingTokens = 8;                  // per SM, from which on the ring is used

struct RingParams {
    RopeParams r;
    uint32_t row_bytes[2];        // of a token: the first run of heads (q, or all of a fused row) and the second (k, or none)
    uint32_t table_bytes;         // of a row of cos or of sin
    uint32_t stage_bytes;
    int stages, consumers;        // consumer threads: lanes of all runs of heads, in whole warps
};
struct RingToken {
    int64_t row;                  // slot in the pool, in tokens, or -1
    int turn, padding;
};

template <typename T, bool HALF, int CACHE, int RUN, bool NORM>
__global__ void __launch_bounds__(kRingThreads + 32, 2) rope_ring_kernel(const __grid_constant__ RingParams rp, int log_lanes) {
    const RopeParams& p = rp.r;
    constexpr bool kCoded = CACHE == CACHE_Q4 || CACHE == CACHE_Q8;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
    __shared__ RingToken info[kMaxStages];
    __shared__ __align__(16) float piece_max[kCoded ? kRingThreads * 2 : 1];
    const int warps = rp.consumers / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < rp.stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, warps);
        }
        mbar_fence_init();
    }
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();
    const int64_t n = (p.T - blockIdx.x + gridDim.x - 1) / gridDim.x;        // tokens of this block
    if (warp == warps) {                                     // ---- producer ----
        int64_t issued = 0;
        bool ok = true;
        int stage = 0;
        uint32_t parity = 1;                                 // of the empty barriers: the first round finds them free
        for (int64_t i0 = 0; i0 < n && ok; i0 += 32) {
            // a lane's token of the next 32
            const int64_t mine = blockIdx.x + (i0 + lane) * gridDim.x;
            const bool live = i0 + lane < n;
            const int pos = live ? p.positions[mine] : 0;
            const int seq = CACHE != NO_CACHE && live && p.sequences ? p.sequences[mine] : (int)mine;
            const bool padding = CACHE != NO_CACHE && seq < 0, in_table = pos >= 0 && pos < p.table_len;
            if (live && !padding && !in_table) atomicMax(&g_device_status, (int)EV_ROPE_POSITION);
            const int64_t row = CACHE != NO_CACHE && live ? cache_row(p, mine, pos, seq, true) : -1;
            const int turn = !padding && in_table;
            for (int k = 0; k < 32 && i0 + k < n; ++k) {
                if (!mbar_wait_bounded(empty + stage, parity, &g_device_status, EV_ROPE_RING, kRingWaitLimit)) {
                    ok = false;
                    break;
                }
                const int at = __shfl_sync(0xFFFFFFFFu, pos, k), turns = __shfl_sync(0xFFFFFFFFu, turn, k), pads = __shfl_sync(0xFFFFFFFFu, (int)padding, k);
                const int64_t slot = __shfl_sync(0xFFFFFFFFu, row, k), t = blockIdx.x + (i0 + k) * gridDim.x;
                if (lane == 0) {
                    info[stage] = {slot, turns, pads};
                    mbar_arrive_expect_tx(full + stage, rp.row_bytes[0] + rp.row_bytes[1] + (turns ? 2 * rp.table_bytes : 0));
                }
                __syncwarp();
                uint8_t* dst = ring + (size_t)stage * rp.stage_bytes;
                const uint32_t rows = rp.row_bytes[0] + rp.row_bytes[1];
                if (lane < 2 && rp.row_bytes[lane] > 0)
                    bulk_g2s(dst + (lane ? rp.row_bytes[0] : 0), reinterpret_cast<const T*>(p.in[lane]) + t * p.in_token[lane], rp.row_bytes[lane], full + stage);
                if ((lane == 2 || lane == 3) && turns)
                    bulk_g2s(dst + rows + (lane == 3 ? rp.table_bytes : 0), (lane == 2 ? p.cos_table : p.sin_table) + (int64_t)at * (p.R / 2), rp.table_bytes, full + stage);
                issued = i0 + k + 1;
                if (++stage == rp.stages) {
                    stage = 0;
                    parity ^= 1u;
                }
            }
        }
        if (!ok)                                             // the consumers gave up: the copies in flight must land before the block ends
            for (int64_t i = max((int64_t)0, issued - rp.stages); i < issued; ++i)
                mbar_wait_bounded(full + i % rp.stages, (uint32_t)(i / rp.stages) & 1u, &g_device_status, EV_ROPE_RING, 1u << 16);
        return;
    }
    // ---- consumers ----
    const int lanes = 1 << log_lanes, l = threadIdx.x & (lanes - 1);
    int run = threadIdx.x >> log_lanes, kind = KIND_Q;
    const bool works = run < p.runs[0] + p.runs[1] + p.runs[2];
    if (run >= p.runs[0]) { run -= p.runs[0]; kind = KIND_K; }
    if (kind == KIND_K && run >= p.runs[1]) { run -= p.runs[1]; kind = KIND_V; }
    const int h0 = run * RUN, count = works ? min(RUN, p.heads[kind] - h0) : 0;
    // first dimensions of the lane's two pieces: interleaved any two, else the u and the v of eight pairs or two pieces behind R
    const int half = p.R / 2, l_turns = half / 8;
    const int d0 = !HALF || l < l_turns ? l * 8 : p.R + (l - l_turns) * 16;
    const int d1 = !HALF ? (l + lanes) * 8 : l < l_turns ? d0 + half : d0 + 8;
    const bool has_turn0 = kind != KIND_V && (HALF ? l < l_turns : d0 < p.R), has_turn1 = kind != KIND_V && (HALF ? l < l_turns : d1 < p.R);
    const int pair0 = HALF ? d0 : d0 / 2, pair1 = HALF ? d0 + 4 : d1 / 2;      // first of four pairs, of c[0..1] and of c[2..3]
    const int first_head = h0 + (kind == KIND_Q ? 0 : kind == KIND_K ? p.heads[0] : p.heads[0] + p.heads[1]);
    const uint32_t rows = rp.row_bytes[0] + rp.row_bytes[1];
    const unsigned group = (lanes == 32 ? 0xFFFFFFFFu : ((1u << lanes) - 1u)) << (lane & ~(lanes - 1));
    const void* weight = NORM && works ? p.weight[kind] : nullptr;
    Pairs w;
    if (NORM && weight != nullptr) {
        float a[8], b[8];
        load_weight8(weight, p.w_dtype, d0, a);
        load_weight8(weight, p.w_dtype, d1, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = 4 * (i & 1);
            w.u[i] = HALF ? pair(a[2 * i], a[2 * i + 1]) : i < 2 ? pair(a[k], a[k + 2]) : pair(b[k], b[k + 2]);
            w.v[i] = HALF ? pair(b[2 * i], b[2 * i + 1]) : i < 2 ? pair(a[k + 1], a[k + 3]) : pair(b[k + 1], b[k + 3]);
        }
    }
    // where the lane reads in a stage, and where it writes: a row that moves with the token, or the token's row of the pool
    const uint32_t at0 = ((uint32_t)first_head * p.D + d0) * 2, at1 = ((uint32_t)first_head * p.D + d1) * 2;
    const uint32_t cos0 = rows + pair0 * 4, cos1 = rows + pair1 * 4;
    const bool to_pool = CACHE != NO_CACHE && kind != KIND_Q;
    T* out = to_pool ? reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(p.codes[kind]) + (int64_t)h0 * p.D * (kCoded ? 1 : 2) / (CACHE == CACHE_Q4 ? 2 : 1))
                     : reinterpret_cast<T*>(p.out[kind]) + blockIdx.x * p.out_token[kind] + (int64_t)h0 * p.out_head[kind];
    const int64_t out_step = to_pool ? (int64_t)p.heads[kind] * p.D : gridDim.x * p.out_token[kind];
    const int64_t head_step = to_pool ? p.D : p.out_head[kind];
    // codes: the groups of the lane's pieces, and its bytes of a head
    float* of_head = piece_max + (kCoded ? (threadIdx.x - l) * 2 : 0);
    const int pieces = p.G / 8, groups = p.D / p.G, g0 = d0 / 8 / pieces * pieces, g1 = d1 / 8 / pieces * pieces;
    const bool in_order = !HALF || p.R == p.D;
    const bool leads0 = d0 % p.G == 0, leads1 = d1 % p.G == 0;
    const int s0_at = d0 / p.G, s1_at = d1 / p.G;
    constexpr int kPerByte = CACHE == CACHE_Q4 ? 2 : 1;
    const int code_head = p.D / kPerByte, code0 = d0 / kPerByte, code1 = d1 / kPerByte;
    const int64_t code_step = (int64_t)p.heads[kind] * code_head;
    const uint8_t* src = ring;
    const float inv_d = 1.0f / (float)p.D;
    int stage = 0;
    uint32_t parity = 0;
    for (int i = 0; i < (int)n; ++i) {
        if (!mbar_wait_bounded(full + stage, parity, &g_device_status, EV_ROPE_RING, kRingWaitLimit)) return;
        const RingToken token = info[stage];
        uint4 x0[RUN], x1[RUN];
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
            x0[j] = x1[j] = make_uint4(0u, 0u, 0u, 0u);
            if (j < count) {
                x0[j] = *reinterpret_cast<const uint4*>(src + at0 + j * p.D * 2);
                x1[j] = *reinterpret_cast<const uint4*>(src + at1 + j * p.D * 2);
            }
        }
        const bool turns0 = token.turn && has_turn0, turns1 = token.turn && has_turn1;
        f32x2 c[4], s[4];
        {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a, e = a, f = a;
            if (turns0) {
                a = *reinterpret_cast<const float4*>(src + cos0);
                b = *reinterpret_cast<const float4*>(src + cos0 + rp.table_bytes);
            }
            if (turns1) {
                e = *reinterpret_cast<const float4*>(src + cos1);
                f = *reinterpret_cast<const float4*>(src + cos1 + rp.table_bytes);
            }
            c[0] = pair(a.x, a.y); c[1] = pair(a.z, a.w); c[2] = pair(e.x, e.y); c[3] = pair(e.z, e.w);
            s[0] = pair(b.x, b.y); s[1] = pair(b.z, b.w); s[2] = pair(f.x, f.y); s[3] = pair(f.z, f.w);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + stage);           // all of the stage is in registers
        src += rp.stage_bytes;
        if (++stage == rp.stages) {
            stage = 0;
            src = ring;
            parity ^= 1u;
        }
        T* row = to_pool ? out + token.row * out_step : out;
        out += to_pool ? 0 : out_step;
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
            Pairs x = unpack<T, !HALF>(x0[j], x1[j]);
            if (NORM && weight != nullptr) {                 // uniform over the lanes of a head
                f32x2 q = mul2(x.u[0], x.u[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) q = fma2(x.u[k], x.u[k], q);
#pragma unroll
                for (int k = 0; k < 4; ++k) q = fma2(x.v[k], x.v[k], q);
                float lo, hi;
                split(q, lo, hi);
                float ss = lo + hi;
                for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor_sync(group, ss, o);
                const float inv = rsqrtf(ss * inv_d + p.eps);      // D is a power of two
                const f32x2 inv2 = pair(inv, inv);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x.u[k] = mul2(mul2(x.u[k], inv2), w.u[k]);
                    x.v[k] = mul2(mul2(x.v[k], inv2), w.v[k]);
                }
            }
            // separately rounded products and one sum, as elementwise operations give them (the sums one by one: a packed product and a
            // packed sum are contracted in spite of their rounding modifiers)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < 2 ? turns0 : turns1) {
                    float uc0, uc1, vs0, vs1, us0, us1, vc0, vc1;
                    split(mul2(x.u[k], c[k]), uc0, uc1);
                    split(mul2(x.v[k], s[k]), vs0, vs1);
                    split(mul2(x.u[k], s[k]), us0, us1);
                    split(mul2(x.v[k], c[k]), vc0, vc1);
                    x.u[k] = pair(__fsub_rn(uc0, vs0), __fsub_rn(uc1, vs1));
                    x.v[k] = pair(__fadd_rn(us0, vc0), __fadd_rn(us1, vc1));
                }
            }
            uint4 y0, y1;
            pack<T, !HALF>(x, y0, y1);
            if (!kCoded || !to_pool) {
                if (j < count && (!to_pool || token.row >= 0)) {
                    if (CACHE != NO_CACHE && token.padding) y0 = y1 = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(row + j * head_step + d0) = y0;
                    *reinterpret_cast<uint4*>(row + j * head_step + d1) = y1;
                }
            } else if (kCoded) {
                // the values as the cache sees them, rounded to T; largest magnitudes by piece, then by group of G/8 pieces in order
                float a[8], b[8];
                bool plain0, plain1;
                float m0 = piece_values<T>(y0, a, plain0), m1 = piece_values<T>(y1, b, plain1);
                if (in_order) {                              // pieces l and l + lanes: the lanes of a group are neighbours
                    if (pieces > lanes) m0 = m1 = fmaxf(m0, m1);
                    for (int o = 1; o < min(pieces, lanes); o <<= 1) {
                        m0 = fmaxf(m0, __shfl_xor_sync(group, m0, o));
                        m1 = fmaxf(m1, __shfl_xor_sync(group, m1, o));
                    }
                } else {
                    __syncwarp(group);
                    of_head[d0 / 8] = m0;
                    of_head[d1 / 8] = m1;
                    __syncwarp(group);
                    for (int k = 0; k < pieces; ++k) {
                        m0 = fmaxf(m0, of_head[g0 + k]);
                        m1 = fmaxf(m1, of_head[g1 + k]);
                    }
                }
                if (j < count && token.row >= 0) {
                    const float q0 = group_scale<CACHE>(m0), q1 = group_scale<CACHE>(m1);
                    uint8_t* codes = reinterpret_cast<uint8_t*>(out) + token.row * code_step + j * code_head;
                    store_codes<CACHE>(a, q0, plain0, codes + code0);
                    store_codes<CACHE>(b, q1, plain1, codes + code1);
                    __half* scales = p.scales[kind] + (token.row * p.heads[kind] + h0 + j) * groups;
                    if (leads0) scales[s0_at] = __float2half_rn(q0);
                    if (leads1) scales[s1_at] = __float2half_rn(q1);
                }
            }
        }
    }
}

// Every other head size, rotary size, group size, stride and alignment: one warp per (token, head), the head in shared memory.
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
    auto scale_of = [&](int g) {
        float m = 0.0f;
        for (int d = g * p.G; d < min(D, (g + 1) * p.G); ++d) m = fmaxf(m, fabsf(y[d]));
        return group_scale<CACHE>(m);
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

bool aligned16(const RopeParams& p) {
    uintptr_t bits = (uintptr_t)p.cos_table | (uintptr_t)p.sin_table;
    for (int i = 0; i < 3; ++i) {
        bits |= (uintptr_t)p.in[i] | (uintptr_t)p.out[i] | (uintptr_t)p.weight[i] | (uintptr_t)p.codes[i];
        bits |= (uintptr_t)((p.in_token[i] | p.in_head[i] | p.out_token[i] | p.out_head[i]) * 2);
    }
    return (bits & 15u) == 0;
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

// Many tokens whose heads are contiguous: the ring kernel; B200Q_ERR_UNSUPPORTED, with nothing launched, for other calls.
template <typename T, int CACHE>
int ring(const RopeParams& params, bool half_layout, int log_lanes, cudaStream_t stream) {
    RingParams rp = {};
    RopeParams& p = rp.r = params;
    const bool fused = CACHE != NO_CACHE;
    const int heads = p.heads[0] + p.heads[1] + p.heads[2], run = (heads << log_lanes) <= kRingThreads ? 1 : 2;
    if (p.T < kRingTokens * sm_count()) return B200Q_ERR_UNSUPPORTED;
    for (int i = 0; i < 2; ++i)
        if (p.heads[i] > 1 && p.in_head[i] != p.D) return B200Q_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i) p.runs[i] = (p.heads[i] + run - 1) / run;
    rp.consumers = (((p.runs[0] + p.runs[1] + p.runs[2]) << log_lanes) + 31) / 32 * 32;
    const uint32_t head_bytes = (uint32_t)p.D * 2;
    rp.row_bytes[0] = (fused ? heads : p.heads[0]) * head_bytes;
    rp.row_bytes[1] = fused ? 0 : p.heads[1] * head_bytes;
    rp.table_bytes = (uint32_t)p.R * 2;
    rp.stage_bytes = (rp.row_bytes[0] + rp.row_bytes[1] + 2 * rp.table_bytes + 127) / 128 * 128;
    rp.stages = (int)std::min<uint32_t>(kMaxStages, kRingBytes / rp.stage_bytes);
    if (rp.consumers > kRingThreads || rp.stages < 3) return B200Q_ERR_UNSUPPORTED;
    const size_t smem = (size_t)rp.stages * rp.stage_bytes;
    const bool norm = p.weight[0] != nullptr || p.weight[1] != nullptr;
    void (*kernel)(const RingParams, int) = half_layout ? (run == 1 ? (norm ? rope_ring_kernel<T, true, CACHE, 1, true> : rope_ring_kernel<T, true, CACHE, 1, false>) : rope_ring_kernel<T, true, CACHE, 2, true>)
                                                        : (run == 1 ? (norm ? rope_ring_kernel<T, false, CACHE, 1, true> : rope_ring_kernel<T, false, CACHE, 1, false>) : rope_ring_kernel<T, false, CACHE, 2, true>);
    // (one value for all calls: two threads may launch the same kernel with different sizes)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes) != cudaSuccess) return B200Q_ERR_LAUNCH;
    return launch(kernel, std::min<int64_t>(p.T, (int64_t)sm_count() * 2), rp.consumers + 32, smem, stream, rp, log_lanes);
}

template <typename T, int CACHE>
int dispatch(RopeParams& p, bool half_layout, cudaStream_t stream) {
    const bool pow2 = (p.D & (p.D - 1)) == 0 && p.D >= 32 && p.D <= 256;
    const bool groups = (CACHE != CACHE_Q4 && CACHE != CACHE_Q8) || (p.G % 8 == 0 && (p.G & (p.G - 1)) == 0 && p.D % p.G == 0);
    if (pow2 && p.R % 16 == 0 && groups && aligned16(p)) {
        int log_lanes = 1;
        while ((16 << log_lanes) < p.D) ++log_lanes;
        const int rc = ring<T, CACHE>(p, half_layout, log_lanes, stream);
        if (rc != B200Q_ERR_UNSUPPORTED) return rc;
        // one head per group of lanes while all of them fit the GPU at once (the shortest chain), else two (RUN)
        const int64_t all = p.T * ((int64_t)p.heads[0] + p.heads[1] + p.heads[2]), per_block = kThreads >> log_lanes;
        const int run = all <= (int64_t)sm_count() * 4 * per_block ? 1 : 2;
        for (int i = 0; i < 3; ++i) p.runs[i] = (p.heads[i] + run - 1) / run;
        const int64_t units = p.T * ((int64_t)p.runs[0] + p.runs[1] + p.runs[2]), blocks = (units + per_block - 1) / per_block;
        if (units <= INT32_MAX) {
            const uint32_t n = (uint32_t)units;
            if (run == 1) {
                if (!half_layout) return launch(rope_heads_kernel<T, INTERLEAVED, CACHE, 1>, blocks, kThreads, 0, stream, p, log_lanes, n);
                if (p.R == p.D) return launch(rope_heads_kernel<T, HALF_WHOLE, CACHE, 1>, blocks, kThreads, 0, stream, p, log_lanes, n);
                return launch(rope_heads_kernel<T, HALF_PART, CACHE, 1>, blocks, kThreads, 0, stream, p, log_lanes, n);
            }
            if (!half_layout) return launch(rope_heads_kernel<T, INTERLEAVED, CACHE, 2>, blocks, kThreads, 0, stream, p, log_lanes, n);
            if (p.R == p.D) return launch(rope_heads_kernel<T, HALF_WHOLE, CACHE, 2>, blocks, kThreads, 0, stream, p, log_lanes, n);
            return launch(rope_heads_kernel<T, HALF_PART, CACHE, 2>, blocks, kThreads, 0, stream, p, log_lanes, n);
        }
    }
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
