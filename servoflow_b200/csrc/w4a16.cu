// w4a16.cu — linear layer with 4-bit weights and group scales, for few rows
// (sfb_w4a16_linear; the 4-bit counterpart of w8a16_gemm.cu).
//
//   Y[m, n] = act( Σ_g s[n, g] · Σ_{k in g} X[m, k] · c[n, k] + bias[n] ) + R[m, n]
//
// Weight rows are the M side of mma.sync m16n8k16 and rows of X its N side, so
// one to eight rows of X cost the same. The codes go from memory to MMA
// fragments in registers: the contraction order inside a group is free, so
// lane (g, t) = (lane / 4, lane % 4) loads the group / 4 consecutive codes it
// needs of channels g and g + 8 with one wide load, and a nibble becomes bf16
// or fp16 exactly with one bit operation and one subtraction (0x4300 | n is
// 128 + n in bf16, 0x6400 | n is 1024 + n in fp16). Products of x and c are
// exact in fp32; a group's sum is scaled in fp32 and added to the row's: no
// rounding to 16 bits anywhere before the output.
//
// A CTA takes 16 output channels and up to 8·NT rows of X; its warps take the
// groups in turn and are joined in shared memory.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sfb {

struct W4Params {
    const void* x;
    const uint8_t* w;
    const void* scale;
    const void *bias, *residual;
    void* y;
    int64_t ldx, ldr, ldy;
    int32_t M, N, K, groups;          // groups = K / group
    int32_t scale_dtype, y_f32;
};

namespace w4 {

constexpr int kWarps = 8;

template <typename T> struct Ops;
template <> struct Ops<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&o)[4]) {
        const __nv_bfloat162 k136 = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), k136);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct Ops<__half> {
    static __device__ __forceinline__ float to_f(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&o)[4]) {
        const __half2 k1032 = __half2half2(__ushort_as_half(0x6408));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
            const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), k1032);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        kv4::mma16816(c, a0, a1, a2, a3, b0, b1);
    }
};

template <int kWords> struct WordsOf;
template <> struct WordsOf<1> { using T = uint32_t; };
template <> struct WordsOf<2> { using T = uint2; };
template <> struct WordsOf<4> { using T = uint4; };

__device__ __forceinline__ float scale_at(const void* s, int dt, int64_t i) {
    if (dt == SFB_F16) return __half2float(static_cast<const __half*>(s)[i]);
    if (dt == SFB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(s)[i]);
    return static_cast<const float*>(s)[i];
}

// G: group; NT: tiles of 8 rows of X; kAct as sfb_w4a16_linear.
template <typename T, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32) w4a16_kernel(const W4Params p, const int act) {
    using O = Ops<T>;
    constexpr int kWords = G / 32;                 // 32-bit words of codes per lane and channel
    using Words = typename WordsOf<kWords>::T;
    __shared__ float red[kWarps][16][NT * 8 + 1];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (NT * 8);
    const int na = min(n0 + g, p.N - 1), nb = min(n0 + g + 8, p.N - 1);   // past the last channel: not stored
    const uint8_t* wa = p.w + static_cast<int64_t>(na) * (p.K / 2) + t * (G / 8);
    const uint8_t* wb = p.w + static_cast<int64_t>(nb) * (p.K / 2) + t * (G / 8);
    const T* x = static_cast<const T*>(p.x);

    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    Words ra{}, rb{};
    if (warp < p.groups) {
        ra = *reinterpret_cast<const Words*>(wa + static_cast<int64_t>(warp) * (G / 2));
        rb = *reinterpret_cast<const Words*>(wb + static_cast<int64_t>(warp) * (G / 2));
    }
    for (int c = warp; c < p.groups; c += kWarps) {
        const Words ca = ra, cb = rb;
        if (c + kWarps < p.groups) {
            ra = *reinterpret_cast<const Words*>(wa + static_cast<int64_t>(c + kWarps) * (G / 2));
            rb = *reinterpret_cast<const Words*>(wb + static_cast<int64_t>(c + kWarps) * (G / 2));
        }
        const float sa = scale_at(p.scale, p.scale_dtype, static_cast<int64_t>(na) * p.groups + c);
        const float sb = scale_at(p.scale, p.scale_dtype, static_cast<int64_t>(nb) * p.groups + c);
        float part[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.f;
#pragma unroll
        for (int q = 0; q < kWords; ++q) {         // 8 codes of a lane: two MMA steps
            uint32_t fa[4], fb[4];
            O::codes(reinterpret_cast<const uint32_t*>(&ca)[q], fa);
            O::codes(reinterpret_cast<const uint32_t*>(&cb)[q], fb);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int m = m0 + j * 8 + g;
                uint4 xv = make_uint4(0, 0, 0, 0);
                if (m < p.M)
                    xv = *reinterpret_cast<const uint4*>(x + m * p.ldx + static_cast<int64_t>(c) * G + t * (G / 4) + q * 8);
                O::mma(part[j], fa[0], fb[0], fa[1], fb[1], xv.x, xv.y);
                O::mma(part[j], fa[2], fb[2], fa[3], fb[3], xv.z, xv.w);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            acc[j][0] = fmaf(sa, part[j][0], acc[j][0]);
            acc[j][1] = fmaf(sa, part[j][1], acc[j][1]);
            acc[j][2] = fmaf(sb, part[j][2], acc[j][2]);
            acc[j][3] = fmaf(sb, part[j][3], acc[j][3]);
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        red[warp][g][j * 8 + 2 * t] = acc[j][0];
        red[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
        red[warp][g + 8][j * 8 + 2 * t] = acc[j][2];
        red[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
    }
    __syncthreads();
    for (int i = tid; i < 16 * NT * 8; i += kWarps * 32) {
        const int ch = i & 15, mm = i >> 4, nn = n0 + ch, m = m0 + mm;
        if (nn >= p.N || m >= p.M) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += red[w][ch][mm];
        if (p.bias != nullptr) v += O::to_f(static_cast<const T*>(p.bias) + nn);
        if (act == 1) v = w8::gelu_tanh(v);
        else if (act == 2) v = v / (1.f + expf(-v));
        if (p.y_f32) {
            if (p.residual != nullptr) v += static_cast<const float*>(p.residual)[m * p.ldr + nn];
            static_cast<float*>(p.y)[m * p.ldy + nn] = v;
        } else {
            if (p.residual != nullptr) v += O::to_f(static_cast<const T*>(p.residual) + m * p.ldr + nn);
            static_cast<T*>(p.y)[m * p.ldy + nn] = O::from_f(v);
        }
    }
}

template <typename T, int G, int NT>
int launch(const W4Params& p, int act, cudaStream_t s) {
    const int64_t bx = (static_cast<int64_t>(p.N) + 15) / 16, by = (static_cast<int64_t>(p.M) + NT * 8 - 1) / (NT * 8);
    if (by > 65535) return SFB_ERR_SHAPE;
    auto kern = w4a16_kernel<T, G, NT>;
    prefer_max_shared(kern);
    return launch_kernel(kern, dim3(static_cast<unsigned>(bx), static_cast<unsigned>(by)), kWarps * 32, 0, s, true, p, act);
}

template <typename T, int G>
int pick_nt(const W4Params& p, int act, cudaStream_t s) {
    if (p.M <= 8) return launch<T, G, 1>(p, act, s);
    if (p.M <= 16) return launch<T, G, 2>(p, act, s);
    if (p.M <= 32) return launch<T, G, 4>(p, act, s);
    return launch<T, G, 9>(p, act, s);
}

template <typename T>
int pick(const W4Params& p, int group, int act, cudaStream_t s) {
    if (group == 32) return pick_nt<T, 32>(p, act, s);
    if (group == 64) return pick_nt<T, 64>(p, act, s);
    return pick_nt<T, 128>(p, act, s);
}

}  // namespace w4

int w4a16_linear_launch(const void* x, int64_t ldx, int32_t x_dtype, const void* w, const void* w_scale,
                        int32_t scale_dtype, int32_t group, const void* bias, const void* residual, int64_t ldr,
                        void* y, int64_t ldy, int32_t y_dtype, int32_t M, int32_t N, int32_t K, int32_t act,
                        cudaStream_t stream) {
    if (M < 0 || N <= 0 || K <= 0) return SFB_ERR_SHAPE;
    if (group != 32 && group != 64 && group != 128) return SFB_ERR_SHAPE;
    if (K % group != 0) return SFB_ERR_SHAPE;
    if (x_dtype != SFB_BF16 && x_dtype != SFB_F16) return SFB_ERR_DTYPE;
    if (y_dtype != x_dtype && y_dtype != SFB_F32) return SFB_ERR_DTYPE;
    if (scale_dtype != SFB_F16 && scale_dtype != SFB_BF16 && scale_dtype != SFB_F32) return SFB_ERR_DTYPE;
    if (act < 0 || act > 2) return SFB_ERR_INVALID;
    if (ldx < K || ldy < N || (residual != nullptr && ldr < N)) return SFB_ERR_SHAPE;
    if (M == 0) return SFB_OK;                     // empty tensors may have no memory
    if (x == nullptr || w == nullptr || w_scale == nullptr || y == nullptr) return SFB_ERR_INVALID;
    auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
    if (!al(x) || !al(w) || ldx % 8 != 0) return SFB_ERR_ALIGN;
    const uintptr_t esz = y_dtype == SFB_F32 ? 4 : 2, ssz = scale_dtype == SFB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(y) % esz || reinterpret_cast<uintptr_t>(residual) % esz ||
        reinterpret_cast<uintptr_t>(bias) % 2 || reinterpret_cast<uintptr_t>(w_scale) % ssz)
        return SFB_ERR_ALIGN;
    if (!is_sm100(device_info())) return SFB_ERR_UNSUPPORTED;
    W4Params p{};
    p.x = x; p.w = static_cast<const uint8_t*>(w); p.scale = w_scale; p.bias = bias; p.residual = residual; p.y = y;
    p.ldx = ldx; p.ldr = ldr; p.ldy = ldy;
    p.M = M; p.N = N; p.K = K; p.groups = K / group;
    p.scale_dtype = scale_dtype; p.y_f32 = y_dtype == SFB_F32 ? 1 : 0;
    return x_dtype == SFB_BF16 ? w4::pick<__nv_bfloat16>(p, group, act, stream) : w4::pick<__half>(p, group, act, stream);
}

}  // namespace sfb
