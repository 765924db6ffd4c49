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
// Both kernels are bound by bytes, if they spend few instructions on each: a row
// of D channels is held by D / 8 lanes, 8 values each (one 16-byte load of a
// 16-bit type, one 32-bit word of codes), 4 lanes make one 32-channel group; a
// warp holds 32 / (D / 8) consecutive tokens of one head, so that its codes are
// one contiguous 128-byte run of the cache, and takes kRuns such runs, loaded
// before the first is worked on; neighbouring warps take neighbouring heads,
// whose source rows are contiguous in a projection's output. Measured (device times,
// calls back to back from a graph): 4 × 4374 tokens of 32 heads of 64 appended 59 µs,
// read back in 16 bits 30 µs (6.1 TB/s, 94 % of a copy's rate); one token of 32
// sessions appended 4.2, read back 1.8 µs. Reading is bound by bytes; appending by the
// issue of its instructions (79 % of the slots for a prompt), a token's by latency.
#include "common.cuh"
#include "sm100_ptx.cuh"

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
    FastDiv tgroups, heads2;       // token groups per session, K and V heads
};

namespace kv4 {

constexpr int kGroup = 32;                       // channels per scale
constexpr int kMoveThreads = 256;
constexpr float kMaxScale = 9344.f;              // 7 · 9344 = 65408, the largest such product in fp16

// (x & mask) | 0x64006400 in one LOP3
template <uint32_t kMask>
__device__ __forceinline__ uint32_t nib_magic(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(kMask), "n"(0x64006400u));
    return r;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// The eight codes of a word as four half2 times s: o[i] = (nibble at 4i, nibble at 16 + 4i).
__device__ __forceinline__ void dequant_word(uint32_t w, __half2 s, uint32_t (&o)[4]) {
    const __half2 k1032 = __half2half2(__ushort_as_half(0x6408));           // 1024 + 8
    const __half2 k16 = __half2half2(__ushort_as_half(0x2c00));             // 1 / 16
    const __half2 k72 = __half2half2(__ushort_as_half(0xd480));             // −(64 + 8)
    const uint32_t w8 = w >> 8;
    o[0] = h2u(__hmul2(__hsub2(u2h(nib_magic<0x000f000fu>(w)), k1032), s));
    o[1] = h2u(__hmul2(__hfma2(u2h(nib_magic<0x00f000f0u>(w)), k16, k72), s));
    o[2] = h2u(__hmul2(__hsub2(u2h(nib_magic<0x000f000fu>(w8)), k1032), s));
    o[3] = h2u(__hmul2(__hfma2(u2h(nib_magic<0x00f000f0u>(w8)), k16, k72), s));
}

constexpr int kRuns = 4;

// Where a warp's work is: session, head (K heads, then V heads), first token.
struct Where { int b, h; int32_t tok; bool is_v, ok; };

template <int D>
__device__ __forceinline__ Where where(const Kv4MoveParams& p) {
    constexpr int kLanes = D / 8, kTok = 32 / kLanes;
    const uint32_t w = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
    const uint32_t wt = p.heads2.div(w), hh = w - wt * p.heads2.d;
    Where r;
    r.ok = w < p.warps;
    r.is_v = hh >= static_cast<uint32_t>(p.c.Hkv);
    r.h = static_cast<int>(hh) - (r.is_v ? p.c.Hkv : 0);
    r.b = static_cast<int>(p.tgroups.div(wt));
    r.tok = static_cast<int>(wt - r.b * p.tgroups.d) * (kTok * kRuns) + (threadIdx.x & 31) / kLanes;
    return r;
}

// fmaxf that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_append_kernel(const Kv4MoveParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int kLanes = D / 8, kTok = 32 / kLanes;
    const Where r = where<D>(p);
    const int sub = threadIdx.x % kLanes;
    if (!r.ok) return;                             // (whole warps)
    const int32_t n = p.len != nullptr ? min(p.seq, p.len[r.b]) : p.seq;
    const int64_t slot0 = static_cast<int64_t>(p.start != nullptr ? p.start[r.b] : p.slot0) + r.tok;
    const int64_t sb = r.is_v ? p.v_st[0] : p.k_st[0], sh = r.is_v ? p.v_st[1] : p.k_st[1], ss = r.is_v ? p.v_st[2] : p.k_st[2];
    const T* src = static_cast<const T*>(r.is_v ? p.v : p.k) + r.b * sb + r.h * sh + r.tok * ss + sub * 8;
    uint8_t* codes = (r.is_v ? p.c.vc : p.c.kc) + r.b * p.c.code_sb + r.h * p.c.code_sh + sub * 4;
    __half* sc = (r.is_v ? p.c.vs : p.c.ks) + r.b * p.c.sc_sb + r.h * p.c.sc_sh + (sub >> 2);
    bool bad = false;
    float x[kRuns][8];
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
        if (r.tok + u * kTok < n) nrope::load8(src + u * kTok * ss, x[u]);
    }
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
        float mx = fabsf(x[u][0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = max_nan(mx, fabsf(x[u][i]));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float s = __half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(mx / 7.f))));
        const bool fits = s <= kMaxScale;          // not for an infinity or a NaN
        uint32_t word = 0x88888888u;
        if (fits && s > 0.f) {
            // x / s correctly rounded, as the division would give it, for eight x and
            // one reciprocal: q = x·y and one residual step q + (x − q·s)·y with y =
            // 1 / s correctly rounded (Markstein, 1990). Then rounded to an integer
            // by adding 1.5·2^23, and four of them combined exactly in fp32.
            const float y = 1.f / s, magic = 12582912.f;
            float half_[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {          // values 2i + e: one 16-bit half of the word
                float acc = 34952.f;               // the + 8 of every nibble: 8·(1 + 16 + 256 + 4096)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float q = x[u][2 * i + e] * y;
                    q = fmaf(fmaf(-q, s, x[u][2 * i + e]), y, q);
                    if (s < 6.1035e-5f) q = fminf(7.f, fmaxf(-7.f, q));   // only a subnormal scale is off by more than 2^-9
                    acc = fmaf((q + magic) - magic, static_cast<float>(1 << (4 * i)), acc);
                }
                half_[e] = acc + 8388608.f;
            }
            word = ptx::prmt(__float_as_uint(half_[0]), __float_as_uint(half_[1]), 0x5410u);
        }
        const int64_t slot = slot0 + u * kTok;
        if (r.tok + u * kTok < n) {
            if (slot >= 0 && slot < p.c.cap) {
                *reinterpret_cast<uint32_t*>(codes + slot * (D / 2)) = word;
                if ((sub & 3) == 0) sc[slot * (D / kGroup)] = fits ? __float2half_rn(s) : __ushort_as_half(0x7fff);
            } else {
                bad = true;
            }
        }
    }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
}

// Four half2 (values 0 1, 2 3, 4 5, 6 7) as 8 values of the output type.
__device__ __forceinline__ void store_halves(__half* p, const uint32_t (&h)[4]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
}
template <typename T>
__device__ __forceinline__ void store_halves(T* p, const uint32_t (&h)[4]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(u2h(h[i]));
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
    nrope::store8(p, x);
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_read_kernel(const Kv4MoveParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int kLanes = D / 8, kTok = 32 / kLanes;
    const Where r = where<D>(p);
    const int sub = threadIdx.x % kLanes;
    T* out = static_cast<T*>(r.is_v ? p.v : p.k);
    if (!r.ok || out == nullptr) return;
    const int64_t slot0 = static_cast<int64_t>(p.slot0) + r.tok;
    const int64_t sb = r.is_v ? p.v_st[0] : p.k_st[0], sh = r.is_v ? p.v_st[1] : p.k_st[1], ss = r.is_v ? p.v_st[2] : p.k_st[2];
    const uint8_t* codes = (r.is_v ? p.c.vc : p.c.kc) + r.b * p.c.code_sb + r.h * p.c.code_sh + slot0 * (D / 2) + sub * 4;
    const __half* sc = (r.is_v ? p.c.vs : p.c.ks) + r.b * p.c.sc_sb + r.h * p.c.sc_sh + slot0 * (D / kGroup) + (sub >> 2);
    out += r.b * sb + r.h * sh + r.tok * ss + sub * 8;
    uint32_t word[kRuns];
    __half s[kRuns];
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
        if (r.tok + u * kTok < p.seq) {
            word[u] = *reinterpret_cast<const uint32_t*>(codes + u * kTok * (D / 2));
            s[u] = sc[u * kTok * (D / kGroup)];
        }
    }
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
        if (r.tok + u * kTok >= p.seq) break;
        uint32_t h[4];
        dequant_word(word[u], __half2half2(s[u]), h);        // exact
        store_halves(out + u * kTok * ss, h);
    }
}

template <typename T>
int launch_move(Kv4MoveParams& p, bool append, cudaStream_t s) {
    const int tok = 32 / (p.c.D / 8);
    const int64_t groups = (static_cast<int64_t>(p.seq) + tok * kRuns - 1) / (tok * kRuns);
    const int64_t warps = static_cast<int64_t>(p.c.B) * groups * 2 * p.c.Hkv;
    if (p.c.Hkv > 0x3fffffff || p.c.B * groups > 0x7fffff00ll || warps > 0x7fffff00ll) return SFB_ERR_SHAPE;
    p.tgroups.set(static_cast<uint32_t>(groups));
    p.heads2.set(static_cast<uint32_t>(2 * p.c.Hkv));
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
    // (slots are counted in 32 bits, up to two blocks of 128 past the last one)
    if (c->batch < 0 || c->heads_kv < 1 || c->capacity < 0 || c->capacity > 0x7ffffe00 || c->capacity % 4 != 0) return SFB_ERR_SHAPE;
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
    if (seq < 0 || seq > 0x7fffff00) return SFB_ERR_SHAPE;
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
