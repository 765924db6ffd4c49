// kv4.cu — the 4-bit K/V cache: quantise new tokens into it (sfb_kv4_append)
// and read slots back in 16 or 32 bits (sfb_kv4_read). The attention over it
// is in kv4_attn.cu.
//
// A value is c·s with a 4-bit code c in [-8, 7] and one fp16 scale s per token,
// head and 32 channels. s is rounded to 8 significant bits (bf16's) before the
// codes are made from it, so c·s (3 more bits) is exact in fp16, the operand
// type of the attention's products: nothing is lost between the cache and the
// tensor cores, and no scale has to be carried into their epilogue.
//
// Both kernels are bound by bytes. A row of D channels is held by D / 8 lanes,
// 8 values each: one 16-byte load of a 16-bit type, one 32-bit word of codes;
// 4 lanes make one 32-channel group. A warp takes 32 / (D / 8) consecutive
// tokens of one head, so that its codes are one contiguous 128-byte run of the
// cache, and neighbouring warps take neighbouring heads, whose source rows are
// contiguous in a projection's output.
#include "common.cuh"

namespace sfb {

struct Kv4Params {
    uint8_t *kc, *vc;
    __half *ks, *vs;
    int64_t code_sb, code_sh;      // bytes
    int64_t sc_sb, sc_sh;          // elements
    int32_t B, Hkv, cap, D;
};

struct Kv4MoveParams {
    Kv4Params c;
    void *k, *v;                   // 16- or 32-bit side (source or destination)
    int64_t k_st[3], v_st[3];      // element strides: batch, head, seq
    int32_t seq, slot0;
    const int32_t *start, *len;
    uint32_t warps;
    int32_t tgroups;               // token groups per session
};

namespace kv4 {

constexpr int kGroup = 32;                       // channels per scale
constexpr int kMoveThreads = 256;
constexpr float kMaxScale = 9344.f;              // 7 · 9344 = 65408, the largest such product in fp16

// Eight codes (c + 8) of one 32-bit word: value 2i at bits 4i, 2i+1 at 16+4i.
__device__ __forceinline__ int nibble_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

struct Where { int b, hh, tok; bool ok; };       // hh: K heads, then V heads

template <int D>
__device__ __forceinline__ Where where(const Kv4MoveParams& p) {
    constexpr int kLanes = D / 8, kTok = 32 / kLanes;
    const uint32_t w = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
    Where r;
    r.ok = w < p.warps;
    const uint32_t heads2 = 2 * p.c.Hkv;
    const uint32_t wt = w / heads2;
    r.hh = static_cast<int>(w - wt * heads2);
    r.b = static_cast<int>(wt / static_cast<uint32_t>(p.tgroups));
    r.tok = static_cast<int>(wt - r.b * p.tgroups) * kTok + (threadIdx.x & 31) / kLanes;
    r.ok = r.ok && r.tok < p.seq;
    return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_append_kernel(const Kv4MoveParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int kLanes = D / 8;
    Where r = where<D>(p);
    const int sub = threadIdx.x % kLanes;
    const bool is_v = r.hh >= p.c.Hkv;
    const int h = is_v ? r.hh - p.c.Hkv : r.hh;
    int64_t slot = 0;
    bool bad = false;
    if (r.ok) {
        if (p.len != nullptr && r.tok >= p.len[r.b]) r.ok = false;
        slot = static_cast<int64_t>(p.start != nullptr ? p.start[r.b] : p.slot0) + r.tok;
        if (r.ok && (slot < 0 || slot >= p.c.cap)) { bad = true; r.ok = false; }
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (r.ok) {
        const int64_t* st = is_v ? p.v_st : p.k_st;
        const T* src = static_cast<const T*>(is_v ? p.v : p.k) + r.b * st[0] + h * st[1] + r.tok * st[2] + sub * 8;
        nrope::load8(src, x);
    }
    // max |x| of the group as an integer: infinities and NaN order above every number
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7fffffffu);
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    float s = __half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(__uint_as_float(mx) / 7.f))));
    const bool fits = mx < 0x7f800000u && s <= kMaxScale;
    uint32_t word = 0x88888888u;
    if (fits && s > 0.f) {
        // x / s correctly rounded, as the division would give it, for eight x and
        // one reciprocal: q = x·y and one residual step q + (x − q·s)·y with y =
        // 1 / s correctly rounded (Markstein, 1990)
        const float y = 1.f / s;
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float q = x[i] * y;
            q = fmaf(fmaf(-q, s, x[i]), y, q);
            const float c = fminf(7.f, fmaxf(-7.f, rintf(q)));
            word |= static_cast<uint32_t>(static_cast<int>(c) + 8) << nibble_shift(i);
        }
    }
    if (r.ok) {
        uint8_t* codes = (is_v ? p.c.vc : p.c.kc) + r.b * p.c.code_sb + h * p.c.code_sh + slot * (D / 2);
        *reinterpret_cast<uint32_t*>(codes + sub * 4) = word;
        if ((sub & 3) == 0) {
            __half* sc = (is_v ? p.c.vs : p.c.ks) + r.b * p.c.sc_sb + h * p.c.sc_sh + slot * (D / kGroup);
            sc[sub >> 2] = fits ? __float2half_rn(s) : __ushort_as_half(0x7fff);
        }
    }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_read_kernel(const Kv4MoveParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int kLanes = D / 8;
    const Where r = where<D>(p);
    const int sub = threadIdx.x % kLanes;
    const bool is_v = r.hh >= p.c.Hkv;
    const int h = is_v ? r.hh - p.c.Hkv : r.hh;
    T* out = static_cast<T*>(is_v ? p.v : p.k);
    if (!r.ok || out == nullptr) return;
    const int64_t slot = static_cast<int64_t>(p.slot0) + r.tok;
    const uint8_t* codes = (is_v ? p.c.vc : p.c.kc) + r.b * p.c.code_sb + h * p.c.code_sh + slot * (D / 2);
    const __half* sc = (is_v ? p.c.vs : p.c.ks) + r.b * p.c.sc_sb + h * p.c.sc_sh + slot * (D / kGroup);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + sub * 4);
    const float s = __half2float(sc[sub >> 2]);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = static_cast<float>(static_cast<int>((word >> nibble_shift(i)) & 15u) - 8) * s;
    const int64_t* st = is_v ? p.v_st : p.k_st;
    nrope::store8(out + r.b * st[0] + h * st[1] + r.tok * st[2] + sub * 8, x);
}

template <typename T>
int launch_move(Kv4MoveParams& p, bool append, cudaStream_t s) {
    const int tok = 32 / (p.c.D / 8);
    p.tgroups = static_cast<int32_t>((static_cast<int64_t>(p.seq) + tok - 1) / tok);
    const int64_t warps = static_cast<int64_t>(p.c.B) * p.tgroups * 2 * p.c.Hkv;
    if (static_cast<int64_t>(p.c.B) * p.tgroups > 0x7fffffff || warps > 0xffffff00ll) return SFB_ERR_SHAPE;
    p.warps = static_cast<uint32_t>(warps);
    const int64_t blocks = (warps * 32 + kMoveThreads - 1) / kMoveThreads;
    auto kern = p.c.D == 64 ? (append ? kv4_append_kernel<T, 64> : kv4_read_kernel<T, 64>)
                            : (append ? kv4_append_kernel<T, 128> : kv4_read_kernel<T, 128>);
    prefer_max_shared(kern);
    return launch_kernel(kern, static_cast<unsigned>(blocks), kMoveThreads, 0, s, true, p);
}

}  // namespace kv4

// Checks a cache and unpacks it; the status of the first thing wrong.
int kv4_cache_check(const sfb_kv4_cache* c, Kv4Params& p) {
    if (c == nullptr) return SFB_ERR_INVALID;
    const bool empty = c->batch == 0 || c->capacity == 0;      // such a cache may have no memory
    if (!empty && (c->k_codes == nullptr || c->v_codes == nullptr || c->k_scale == nullptr || c->v_scale == nullptr))
        return SFB_ERR_INVALID;
    if (c->head_dim != 64 && c->head_dim != 128) return SFB_ERR_SHAPE;
    if (c->batch < 0 || c->heads_kv < 1 || c->capacity < 0 || c->capacity % 4 != 0) return SFB_ERR_SHAPE;
    auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
    if (!al(c->k_codes) || !al(c->v_codes) || !al(c->k_scale) || !al(c->v_scale)) return SFB_ERR_ALIGN;
    if (c->code_stride[0] % 16 || c->code_stride[1] % 16 || c->scale_stride[0] % 8 || c->scale_stride[1] % 8)
        return SFB_ERR_ALIGN;
    p.kc = static_cast<uint8_t*>(c->k_codes); p.vc = static_cast<uint8_t*>(c->v_codes);
    p.ks = static_cast<__half*>(c->k_scale);  p.vs = static_cast<__half*>(c->v_scale);
    p.code_sb = c->code_stride[0]; p.code_sh = c->code_stride[1];
    p.sc_sb = c->scale_stride[0];  p.sc_sh = c->scale_stride[1];
    p.B = c->batch; p.Hkv = c->heads_kv; p.cap = c->capacity; p.D = c->head_dim;
    return SFB_OK;
}

// The 16- or 32-bit side of a move: pointer and strides of 16 bytes' multiples.
static int kv4_side(const void* x, const int64_t* st, int32_t dtype, void** px, int64_t* pst) {
    *px = const_cast<void*>(x);
    if (x == nullptr) return SFB_OK;
    if (st == nullptr) return SFB_ERR_INVALID;
    const int vec = dtype == SFB_F32 ? 4 : 8;
    if ((reinterpret_cast<uintptr_t>(x) & 15u) || st[0] % vec || st[1] % vec || st[2] % vec) return SFB_ERR_ALIGN;
    for (int i = 0; i < 3; ++i) pst[i] = st[i];
    return SFB_OK;
}

static int kv4_move(Kv4MoveParams& p, int32_t dtype, bool append, cudaStream_t s) {
    if (!is_sm100(device_info())) return SFB_ERR_UNSUPPORTED;
    if (dtype == SFB_BF16) return kv4::launch_move<__nv_bfloat16>(p, append, s);
    if (dtype == SFB_F16) return kv4::launch_move<__half>(p, append, s);
    return kv4::launch_move<float>(p, append, s);
}

int kv4_append_launch(const sfb_kv4_cache* cache, const void* k, const int64_t* k_st, const void* v,
                      const int64_t* v_st, int32_t dtype, int32_t seq, const int32_t* start, int32_t slot0,
                      const int32_t* len, cudaStream_t s) {
    Kv4MoveParams p{};
    SFB_TRY(kv4_cache_check(cache, p.c));
    if (dtype != SFB_F32 && dtype != SFB_F16 && dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (seq < 0) return SFB_ERR_SHAPE;
    // without per-session starts the slots are known here
    if (start == nullptr && (slot0 < 0 || static_cast<int64_t>(slot0) + seq > cache->capacity)) return SFB_ERR_SHAPE;
    if (p.c.B == 0 || seq == 0) return SFB_OK;
    if (k == nullptr || v == nullptr) return SFB_ERR_INVALID;
    SFB_TRY(kv4_side(k, k_st, dtype, &p.k, p.k_st));
    SFB_TRY(kv4_side(v, v_st, dtype, &p.v, p.v_st));
    p.seq = seq; p.slot0 = slot0; p.start = start; p.len = len;
    return kv4_move(p, dtype, true, s);
}

int kv4_read_launch(const sfb_kv4_cache* cache, void* k, const int64_t* k_st, void* v, const int64_t* v_st,
                    int32_t dtype, int32_t slot0, int32_t seq, cudaStream_t s) {
    Kv4MoveParams p{};
    SFB_TRY(kv4_cache_check(cache, p.c));
    if (dtype != SFB_F32 && dtype != SFB_F16 && dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (seq < 0 || slot0 < 0 || static_cast<int64_t>(slot0) + seq > cache->capacity) return SFB_ERR_SHAPE;
    if (p.c.B == 0 || seq == 0) return SFB_OK;
    if (k == nullptr && v == nullptr) return SFB_ERR_INVALID;
    SFB_TRY(kv4_side(k, k_st, dtype, &p.k, p.k_st));
    SFB_TRY(kv4_side(v, v_st, dtype, &p.v, p.v_st));
    p.seq = seq; p.slot0 = slot0;
    return kv4_move(p, dtype, false, s);
}

}  // namespace sfb
