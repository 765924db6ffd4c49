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
// Bound: bytes (each value read once and written once), if few instructions go
// with them. A head is held by D / 8 lanes, 8 values (one 16-byte load of a
// 16-bit type) each, so the mean is log2(lanes) shuffles, and the rotation's
// partner value of the half-split form is one shuffle away (pairs (i, i + rot/2)
// with rot % 16 == 0 keep the same slot of another lane; the interleaved form's
// partner is in the lane). A thread takes kHeads neighbouring heads of one token:
// they share its position's cos / sin values (8 + 8 fp32 loads beside 8 16-bit
// ones) and the index arithmetic. Blocks of q come before blocks of k, so that
// which of the two a thread works on costs nothing per head.
// Measured (device times, calls back to back from a graph; an eager call costs the host
// 18 µs): 32 × 67 tokens of 32 + 32 heads of 64, 7.9 µs; 2 × 4374 tokens of 32 +
// 8 heads of 128, 35.1 µs (5.2 TB/s, 79 % of a copy's rate); one token 1.5 µs.
#include "common.cuh"

namespace sfb {

// Division of n < 2^31 by a constant (Granlund and Montgomery, 1994).
struct FastDiv {
    uint32_t mul, shift, d;
    void set(uint32_t x) {
        d = x; shift = 0;
        while ((1u << shift) < x) ++shift;
        mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - x)) / x + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct NormRopeSide {
    const void* x;
    void* out;
    const void* w;
    int64_t st[3], so[3];                             // element strides: batch, head, seq
    int32_t heads;
    FastDiv chunks;                                   // groups of kHeads heads
};

struct NormRopeParams {
    NormRopeSide side[2];                             // q, k
    const float *cos_t, *sin_t;
    const int32_t* pos;
    int64_t pos_sb;
    FastDiv S;
    int32_t table_len, D, rot, norm;
    uint32_t tokens, blocks_q;
    float eps, inv_d;                                 // 1 / D
};

namespace nrope {

constexpr int kThreads = 128;

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

// kLanes: lanes per head (8, 16 or 32; D / 8 of them hold values); kHeads: heads
// per thread; kRot: 0 no rotation, 1 pairs (i, i + rot/2), 2 pairs (2i, 2i+1).
template <typename T, int kLanes, int kHeads, int kRot>
__global__ void __launch_bounds__(kThreads)
norm_rope_kernel(const NormRopeParams p) {
    pdl_trigger();
    const bool is_k = blockIdx.x >= p.blocks_q;
    const NormRopeSide& sd = p.side[is_k ? 1 : 0];
    const uint32_t unit = (blockIdx.x - (is_k ? p.blocks_q : 0)) * (kThreads / kLanes) + threadIdx.x / kLanes;
    const int d0 = (threadIdx.x % kLanes) * 8;
    const uint32_t tok = sd.chunks.div(unit), h0 = (unit - tok * sd.chunks.d) * kHeads;
    const bool in_range = tok < p.tokens;             // whole warps take the shuffles below
    const uint32_t b = p.S.div(in_range ? tok : 0), s = (in_range ? tok : 0) - b * p.S.d;
    const bool act = in_range && d0 < p.D;
    const int nh = act ? min(kHeads, sd.heads - static_cast<int>(h0)) : 0;
    const int64_t hs = sd.st[1], ho = sd.so[1];
    const T* src = static_cast<const T*>(sd.x) + b * sd.st[0] + h0 * hs + s * sd.st[2] + d0;
    pdl_wait();
    const int64_t pos = kRot != 0 && p.pos != nullptr ? p.pos[b * p.pos_sb + s] : static_cast<int64_t>(s);
    float x[kHeads][8];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
        if (j < nh) load8(src + j * hs, x[j]);
    }
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = 1.f;
    if (sd.w != nullptr && act) load8(static_cast<const T*>(sd.w) + d0, g);
    // the token's angles: 8 (half-split) or 4 (interleaved) pairs for this lane. Lanes
    // past the rotated channels take no part: a product with a sine of 0 would make
    // NaN of an infinity there, and of its neighbour. (Left out by selecting the result
    // where pairs are interleaved, by a branch where halves are paired. Exchanged,
    // 2 × 4374 tokens of 40 heads took 35.9 µs for 35.1, 32 × 67 tokens 8.5 for 7.8.)
    float c[8], sn[8];
    bool bad = false;
    const bool first = d0 < p.rot / 2, turns = d0 < p.rot;
    if constexpr (kRot != 0) {
        bad = pos < 0 || pos >= p.table_len;
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = sn[i] = 0.f;
        if (turns && !bad) {
            const int64_t base = pos * (p.rot / 2);
            if constexpr (kRot == 2) {
                const float4 cc = *reinterpret_cast<const float4*>(p.cos_t + base + d0 / 2);
                const float4 ss = *reinterpret_cast<const float4*>(p.sin_t + base + d0 / 2);
                c[0] = cc.x; c[1] = cc.y; c[2] = cc.z; c[3] = cc.w;
                sn[0] = ss.x; sn[1] = ss.y; sn[2] = ss.z; sn[3] = ss.w;
            } else {
                const int i0 = first ? d0 : d0 - p.rot / 2;
                load8(p.cos_t + base + i0, c);
                load8(p.sin_t + base + i0, sn);
#pragma unroll
                for (int i = 0; i < 8; ++i) sn[i] = first ? -sn[i] : sn[i];      // a·cos − b·sin, b·cos + a·sin
            }
        }
    }
    // the lane of the pair's other half (this one where nothing is rotated)
    const int lane = threadIdx.x & 31, hop = p.rot / 16;
    const int peer = turns ? (first ? lane + hop : lane - hop) : lane;
    T* dst = static_cast<T*>(sd.out) + b * sd.so[0] + h0 * ho + s * sd.so[2] + d0;
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        float (&f)[8] = x[j];
        if (p.norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss = fmaf(f[2 * i], f[2 * i], fmaf(f[2 * i + 1], f[2 * i + 1], ss));
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(fmaf(ss, p.inv_d, p.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * g[i];
        }
        if constexpr (kRot == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = f[2 * i], bb = f[2 * i + 1];
                f[2 * i]     = turns ? a * c[i] - bb * sn[i] : a;
                f[2 * i + 1] = turns ? bb * c[i] + a * sn[i] : bb;
            }
        } else if constexpr (kRot == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float o = __shfl_sync(0xffffffffu, f[i], peer);
                if (turns) f[i] = f[i] * c[i] + o * sn[i];
            }
        }
        if (j < nh && !bad) store8(dst + j * ho, f);
    }
    if (kRot != 0 && act && bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
}

template <typename T, int kLanes, int kHeads, int kRot>
int launch(NormRopeParams& p, cudaStream_t s) {
    int64_t blocks[2];
    for (int i = 0; i < 2; ++i) {
        NormRopeSide& sd = p.side[i];
        const uint32_t chunks = static_cast<uint32_t>((sd.heads + kHeads - 1) / kHeads);
        const int64_t units = static_cast<int64_t>(p.tokens) * chunks;
        if (units >= 0x7fffff00ll) return SFB_ERR_SHAPE;
        sd.chunks.set(std::max(chunks, 1u));
        blocks[i] = (units * kLanes + kThreads - 1) / kThreads;
    }
    if (blocks[0] + blocks[1] > 0x7fffffff) return SFB_ERR_SHAPE;
    p.blocks_q = static_cast<uint32_t>(blocks[0]);
    auto kern = norm_rope_kernel<T, kLanes, kHeads, kRot>;
    prefer_max_shared(kern);
    return launch_kernel(kern, static_cast<unsigned>(blocks[0] + blocks[1]), kThreads, 0, s, true, p);
}

template <typename T, int kLanes>
int pick_rot(NormRopeParams& p, bool inter, cudaStream_t s) {
    // Four heads per thread once one per thread would be 1536 threads an SM: four
    // loads in flight each, the angles' loads and the index arithmetic a quarter.
    // Below that a call is latency. 64 heads of 64, one and four heads per thread: 4
    // × 67 tokens 2.7 and 3.4 µs, 32 × 16 tokens 3.6 and 3.0, 32 × 67 11.2 and 7.9.
    const int64_t one = static_cast<int64_t>(p.tokens) * (p.side[0].heads + p.side[1].heads) * kLanes;
    const bool many = one >= static_cast<int64_t>(std::max(device_info().num_sms, 1)) * 1536;
    if (p.rot == 0) return many ? launch<T, kLanes, 4, 0>(p, s) : launch<T, kLanes, 1, 0>(p, s);
    if (inter) return many ? launch<T, kLanes, 4, 2>(p, s) : launch<T, kLanes, 1, 2>(p, s);
    return many ? launch<T, kLanes, 4, 1>(p, s) : launch<T, kLanes, 1, 1>(p, s);
}

template <typename T>
int pick(NormRopeParams& p, bool inter, cudaStream_t s) {
    if (p.D <= 64) return pick_rot<T, 8>(p, inter, s);
    if (p.D <= 128) return pick_rot<T, 16>(p, inter, s);
    return pick_rot<T, 32>(p, inter, s);
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
    NormRopeSide &q = p.side[0], &k = p.side[1];
    q.x = a.q; q.out = a.q_out; q.w = a.q_weight; q.heads = H;
    k.x = a.k; k.out = a.k_out; k.w = a.k_weight; k.heads = Hkv;
    for (int i = 0; i < 3; ++i) {
        q.st[i] = a.q_stride[i]; q.so[i] = a.q_out_stride[i];
        k.st[i] = a.k_stride[i]; k.so[i] = a.k_out_stride[i];
    }
    p.cos_t = a.cos_table; p.sin_t = a.sin_table;
    p.pos = a.positions; p.pos_sb = a.pos_stride_b;
    p.table_len = a.table_len;
    p.S.set(static_cast<uint32_t>(a.seq)); p.D = a.head_dim; p.rot = a.rotary_dim;
    p.norm = a.norm ? 1 : 0; p.eps = a.eps; p.inv_d = 1.f / static_cast<float>(a.head_dim);
    const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq;
    if (tokens > 0x7fffff00ll) return SFB_ERR_SHAPE;
    p.tokens = static_cast<uint32_t>(tokens);
    const bool inter = a.interleaved != 0;
    if (a.dtype == SFB_BF16) return nrope::pick<__nv_bfloat16>(p, inter, s);
    if (a.dtype == SFB_F16) return nrope::pick<__half>(p, inter, s);
    return nrope::pick<float>(p, inter, s);
}

}  // namespace sfb
