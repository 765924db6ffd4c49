// norm_rope.cu — RMS norm of the query and key heads with the position
// rotation in the same pass (sfb_qk_norm_rope).
//
//   y = x / sqrt(mean(x²) + eps) · w            per head of D channels
//   (a, b) → (a·cos − b·sin, b·cos + a·sin)     per pair of the first `rot` channels
//
// The two steps the reference runs as separate passes over Q and K
// (qk-norm, src/models/rdt1b/dit_block.cu:185-196 → norm.cuh:89-122) are one
// here: fp32 from the load to the single rounding of the store.
//
// Bound: bytes (each value read once and written once). A head is held by
// D / 8 lanes, 8 values (one 16-byte load of a 16-bit type) each, so the mean
// is log2(lanes) shuffles, and the rotation's partner value of the half-split
// form is one shuffle away (pairs (i, i + rot/2) with rot % 16 == 0 keep the
// same slot of another lane; the interleaved form's partner is in the lane).
// A thread takes up to kHeads heads of one token: they share the token's
// cos / sin values, whose loads would otherwise be four times the data's
// (8 + 8 fp32 values per 8 16-bit ones).
#include "common.cuh"

namespace sfb {

struct NormRopeParams {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_st[3], qo_st[3], k_st[3], ko_st[3];     // element strides: batch, head, seq
    const void *q_w, *k_w;
    const float *cos_t, *sin_t;
    const int32_t* pos;
    int64_t pos_sb;
    int32_t table_len, S, H, Hkv, D, rot, norm;
    int32_t chunks;                                   // threads (of a head's lane) per token
    uint32_t tokens;
    float eps, inv_d;                                 // 1 / D
};

namespace nrope {

constexpr int kThreads = 256;

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) { const float2 f = __bfloat1622float2(h[k]); v[2 * k] = f.x; v[2 * k + 1] = f.y; }
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) { const float2 f = __half22float2(h[k]); v[2 * k] = f.x; v[2 * k + 1] = f.y; }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// kLanes: lanes per head (8, 16 or 32; D / 8 of them hold values);
// kHeads: heads per thread; kInter: pairs (2i, 2i+1) instead of (i, i + rot/2).
template <typename T, int kLanes, int kHeads, bool kInter>
__global__ void __launch_bounds__(kThreads)
norm_rope_kernel(const NormRopeParams p) {
    pdl_trigger();
    pdl_wait();
    const uint32_t unit = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
    const int sub = threadIdx.x % kLanes;
    const uint32_t tok = unit / static_cast<uint32_t>(p.chunks);
    const int chunk = static_cast<int>(unit - tok * p.chunks);
    const bool in_range = tok < p.tokens;             // whole warps take the shuffles below
    const uint32_t bi = in_range ? tok / static_cast<uint32_t>(p.S) : 0;
    const int64_t b = bi, s = in_range ? tok - bi * p.S : 0;
    const int64_t pos = in_range && p.rot > 0 && p.pos != nullptr ? p.pos[b * p.pos_sb + s] : s;
    const int d0 = sub * 8;
    const bool act = in_range && d0 < p.D;
    const int heads = p.H + p.Hkv;

    float x[kHeads][8];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int h = chunk + j * p.chunks;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
        if (act && h < heads) {
            const T* src = h < p.H
                ? static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + s * p.q_st[2]
                : static_cast<const T*>(p.k) + b * p.k_st[0] + (h - p.H) * p.k_st[1] + s * p.k_st[2];
            load8(src + d0, x[j]);
        }
    }
    // the weights of this lane's channels (q's and k's differ only by head)
    float gq[8], gk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) gq[i] = gk[i] = 1.f;
    if (p.norm && act) {
        if (p.q_w != nullptr && chunk < p.H) load8(static_cast<const T*>(p.q_w) + d0, gq);
        if (p.k_w != nullptr && chunk + (kHeads - 1) * p.chunks >= p.H) load8(static_cast<const T*>(p.k_w) + d0, gk);
    }
    // the token's angles: 8 (half-split) or 4 (interleaved) pairs for this lane
    float c[8], sn[8];
    bool bad = false;
    const bool rotates = p.rot > 0 && d0 < p.rot;
    if (p.rot > 0 && in_range) {
        bad = pos < 0 || pos >= p.table_len;
        if (rotates && !bad) {
            const int64_t base = pos * (p.rot / 2);
            if constexpr (kInter) {
                const float4 cc = *reinterpret_cast<const float4*>(p.cos_t + base + d0 / 2);
                const float4 ss = *reinterpret_cast<const float4*>(p.sin_t + base + d0 / 2);
                c[0] = cc.x; c[1] = cc.y; c[2] = cc.z; c[3] = cc.w;
                sn[0] = ss.x; sn[1] = ss.y; sn[2] = ss.z; sn[3] = ss.w;
            } else {
                const int i0 = d0 < p.rot / 2 ? d0 : d0 - p.rot / 2;
                load8(p.cos_t + base + i0, c);
                load8(p.sin_t + base + i0, sn);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int h = chunk + j * p.chunks;
        const bool have = act && h < heads;
        float (&f)[8] = x[j];
        if (p.norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss = fmaf(f[2 * i], f[2 * i], fmaf(f[2 * i + 1], f[2 * i + 1], ss));
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(fmaf(ss, p.inv_d, p.eps));
            const bool is_q = h < p.H;
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * (is_q ? gq[i] : gk[i]);
        }
        if (p.rot > 0) {
            if constexpr (kInter) {
                if (rotates && !bad) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = f[2 * i], bb = f[2 * i + 1];
                        f[2 * i]     = a * c[i] - bb * sn[i];
                        f[2 * i + 1] = bb * c[i] + a * sn[i];
                    }
                }
            } else {
                const bool first = d0 < p.rot / 2;
                const int lane = threadIdx.x & 31, hop = p.rot / 16;
                const int peer = rotates ? (first ? lane + hop : lane - hop) : lane;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float o = __shfl_sync(0xffffffffu, f[i], peer);
                    if (rotates && !bad) f[i] = first ? f[i] * c[i] - o * sn[i] : f[i] * c[i] + o * sn[i];
                }
            }
        }
        if (have && !bad) {
            T* dst = h < p.H
                ? static_cast<T*>(p.q_out) + b * p.qo_st[0] + h * p.qo_st[1] + s * p.qo_st[2]
                : static_cast<T*>(p.k_out) + b * p.ko_st[0] + (h - p.H) * p.ko_st[1] + s * p.ko_st[2];
            store8(dst + d0, f);
        }
    }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
}

template <typename T, int kLanes, bool kInter>
int launch(NormRopeParams& p, cudaStream_t s) {
    // Four heads per thread once that still leaves half the GPU's threads busy:
    // four loads in flight each, the angles' loads a quarter. One head per
    // thread below that, where a call is latency.
    const int heads = p.H + p.Hkv;
    const int64_t one = static_cast<int64_t>(p.tokens) * heads * kLanes;
    const bool many = one >= static_cast<int64_t>(std::max(device_info().num_sms, 1)) * 1024 * 4;
    const int per = many ? 4 : 1;
    p.chunks = (heads + per - 1) / per;
    const int64_t units = static_cast<int64_t>(p.tokens) * p.chunks, blocks = (units * kLanes + kThreads - 1) / kThreads;
    if (units > 0xffffff00ll || blocks > 0x7fffffff) return SFB_ERR_SHAPE;
    auto kern = many ? norm_rope_kernel<T, kLanes, 4, kInter> : norm_rope_kernel<T, kLanes, 1, kInter>;
    prefer_max_shared(kern);
    return launch_kernel(kern, static_cast<unsigned>(blocks), kThreads, 0, s, true, p);
}

template <typename T>
int pick(NormRopeParams& p, bool inter, cudaStream_t s) {
    if (p.D <= 64)
        return inter ? launch<T, 8, true>(p, s) : launch<T, 8, false>(p, s);
    if (p.D <= 128)
        return inter ? launch<T, 16, true>(p, s) : launch<T, 16, false>(p, s);
    return inter ? launch<T, 32, true>(p, s) : launch<T, 32, false>(p, s);
}

}  // namespace nrope

int qk_norm_rope_launch(const sfb_norm_rope_args& a, cudaStream_t s) {
    if (a.batch == 0 || a.seq == 0) return SFB_OK;             // empty tensors may have no memory
    if ((a.q == nullptr) != (a.q_out == nullptr) || (a.k == nullptr) != (a.k_out == nullptr)) return SFB_ERR_INVALID;
    if (a.q == nullptr && a.k == nullptr) return SFB_ERR_INVALID;
    const int H = a.q != nullptr ? a.heads : 0, Hkv = a.k != nullptr ? a.heads_kv : 0;
    if (a.batch < 0 || a.seq < 0 || H < 0 || Hkv < 0) return SFB_ERR_SHAPE;
    if (a.dtype != SFB_F32 && a.dtype != SFB_F16 && a.dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8 != 0) return SFB_ERR_SHAPE;
    if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 16 != 0) return SFB_ERR_SHAPE;
    if (a.rotary_dim > 0 && (a.cos_table == nullptr || a.sin_table == nullptr)) return SFB_ERR_INVALID;
    if (a.rotary_dim > 0 && a.table_len < 0) return SFB_ERR_SHAPE;
    if (H + Hkv == 0) return SFB_OK;
    const int vec = a.dtype == SFB_F32 ? 4 : 8;
    auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    auto st = [&](const int64_t* x) { return x[0] % vec == 0 && x[1] % vec == 0 && x[2] % vec == 0; };
    if (H > 0 && !(al(a.q) && al(a.q_out) && st(a.q_stride) && st(a.q_out_stride))) return SFB_ERR_ALIGN;
    if (Hkv > 0 && !(al(a.k) && al(a.k_out) && st(a.k_stride) && st(a.k_out_stride))) return SFB_ERR_ALIGN;
    if (!al(a.q_weight) || !al(a.k_weight) || !al(a.cos_table) || !al(a.sin_table)) return SFB_ERR_ALIGN;
    if (!is_sm100(device_info())) return SFB_ERR_UNSUPPORTED;
    NormRopeParams p{};
    p.q = a.q; p.k = a.k; p.q_out = a.q_out; p.k_out = a.k_out;
    for (int i = 0; i < 3; ++i) {
        p.q_st[i] = a.q_stride[i]; p.qo_st[i] = a.q_out_stride[i];
        p.k_st[i] = a.k_stride[i]; p.ko_st[i] = a.k_out_stride[i];
    }
    p.q_w = a.q_weight; p.k_w = a.k_weight;
    p.cos_t = a.cos_table; p.sin_t = a.sin_table;
    p.pos = a.positions; p.pos_sb = a.pos_stride_b;
    p.table_len = a.table_len;
    p.S = a.seq; p.H = H; p.Hkv = Hkv; p.D = a.head_dim; p.rot = a.rotary_dim;
    p.norm = a.norm ? 1 : 0; p.eps = a.eps; p.inv_d = 1.f / static_cast<float>(a.head_dim);
    const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq;
    if (tokens > 0x7fffffff) return SFB_ERR_SHAPE;
    p.tokens = static_cast<uint32_t>(tokens);
    const bool inter = a.interleaved != 0;
    if (a.dtype == SFB_BF16) return nrope::pick<__nv_bfloat16>(p, inter, s);
    if (a.dtype == SFB_F16) return nrope::pick<__half>(p, inter, s);
    return nrope::pick<float>(p, inter, s);
}

}  // namespace sfb
