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
// Two kernels. Up to 16 rows are bound by the weights' bytes, if few instructions
// go with them (a 1 KB chunk of 16 channels is 96 for the codes and MMAs alone): a
// CTA takes 16 or 32 channels, its eight warps chunks of 128 inputs by turns, with
// everything of a warp's next chunk (codes, scales, X) in flight while it works on
// one, in two sets of registers by turns. More rows are bound by X, which every
// CTA reads from L2: a CTA takes 64 channels (32 when those are too few CTAs) and
// 8·NT rows, X goes through a ring of shared memory that the warps of the channel
// tiles share, and the warps left over split the inputs.
//
// Measured (device times, calls back to back from a graph; an eager call costs the host
// 12 µs): one row of 16384 × 8192, groups of 128, 26.6 µs (2.6 TB/s of codes and
// scales); one of 2048² 3.0; 8 of 8192² 19.2 (21.7 with other buffers); 67 of 6144 × 2048
// 20.1; 2144 of 2048² 120. The int8 layer takes 57.8, 8.6, 32.3, 12.7 and 22.2 µs: this
// one is faster up to 16 rows; 24 take 11.6 and 11.6 µs (6144 × 2048), 44.5 and 32.3
// (8192²). What bounds few rows is the loads' latency and the issue of instructions
// together, 165 a KB of codes in 43 % of the slots: more bytes in flight (warp-private
// rings of asynchronous copies, 4 stages deep, 204 a KB) gave 24.3, 3.8 and 20.8 µs for
// the first three. More rows are bound by X from L2, the conversion of the codes by
// every warp for each 72 rows and mma.sync's rate, 67 of 6144 × 2048 also by 96 CTAs for
// 148 SMs.
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

// (x & 0x000f000f) | kMagic in one LOP3 (two constants: the compiler takes two)
template <uint32_t kMagic>
__device__ __forceinline__ uint32_t nib_or(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(0x000f000fu), "n"(kMagic));
    return r;
}

template <typename T> struct Ops;
template <> struct Ops<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&o)[4]) {
        const __nv_bfloat162 k136 = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = nib_or<0x43004300u>(w >> (4 * i));
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), k136);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
};
template <> struct Ops<__half> {
    static __device__ __forceinline__ float to_f(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&o)[4]) {
        const __half2 k1032 = __half2half2(__ushort_as_half(0x6408));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = nib_or<0x64006400u>(w >> (4 * i));
            const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), k1032);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
        kv4::mma16816(c, a0, a1, a2, a3, b0, b1);
    }
    static __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
};

__device__ __forceinline__ float scale_at(const void* s, int dt, int64_t i) {
    if (dt == SFB_F16) return __half2float(static_cast<const __half*>(s)[i]);
    if (dt == SFB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(s)[i]);
    return static_cast<const float*>(s)[i];
}

constexpr int kChunk = 128;                        // inputs of a chunk
constexpr int kThreads = kWarps * 32;

// A lane's codes of a chunk are four words of 8. Inside a chunk the inputs are
// dealt out in blocks of 64 (of 32 for groups of 32): lane t has a quarter of each
// block, word w of the four belongs to block w / kQ. Groups are whole blocks.
__host__ __device__ constexpr int block_of(int G) { return G < 64 ? 32 : 64; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes_in) {
    // 16 bytes, of which bytes_in are read and the rest zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes_in) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The join and the epilogue. red: [parts][channels][rows + 1] fp32 sums. A thread
// keeps one channel; its bias and residuals are loaded (`before`) ahead of the
// barrier that the sums wait for.
template <typename T, int kChannels, int kRows, int kThr, int kPartSums>
struct Epilogue {
    static constexpr int kStep = kThr / kChannels, kIt = (kRows + kStep - 1) / kStep;
    static_assert(kThr % kChannels == 0, "a thread keeps its channel");
    int nn, mm0, m0;
    float bias, res[kIt];

    __device__ __forceinline__ void before(const W4Params& p, int n0, int m0_) {
        using O = Ops<T>;
        nn = n0 + threadIdx.x % kChannels;
        mm0 = threadIdx.x / kChannels;
        m0 = m0_;
        bias = p.bias != nullptr && nn < p.N ? O::to_f(static_cast<const T*>(p.bias) + nn) : 0.f;
#pragma unroll
        for (int i = 0; i < kIt; ++i) {
            const int mm = mm0 + i * kStep;
            const int64_t m = m0 + mm;
            res[i] = 0.f;
            if (p.residual != nullptr && nn < p.N && mm < kRows && m < p.M)
                res[i] = p.y_f32 ? static_cast<const float*>(p.residual)[m * p.ldr + nn]
                                 : O::to_f(static_cast<const T*>(p.residual) + m * p.ldr + nn);
        }
    }
    __device__ __forceinline__ void after(const W4Params& p, int act, const float* red) {
        if (nn >= p.N) return;
        const int ch = threadIdx.x % kChannels;
#pragma unroll
        for (int i = 0; i < kIt; ++i) {
            const int mm = mm0 + i * kStep;
            const int64_t m = m0 + mm;
            if (mm >= kRows || m >= p.M) break;
            float v = bias;
#pragma unroll
            for (int w = 0; w < kPartSums; ++w) v += red[(w * kChannels + ch) * (kRows + 1) + mm];
            if (act == 1) v = w8::gelu_tanh(v);
            else if (act == 2) v = v / (1.f + expf(-v));
            v += res[i];
            if (p.y_f32) static_cast<float*>(p.y)[m * p.ldy + nn] = v;
            else static_cast<T*>(p.y)[m * p.ldy + nn] = Ops<T>::from_f(v);
        }
    }
};

// part (+)= one word's products for every tile of 8 rows; the first word of a
// group starts the sums.
template <typename T, int NT>
__device__ __forceinline__ void word_mma(float (&part)[NT][4], uint32_t wa, uint32_t wb, const uint4 (&x)[NT], bool first) {
    using O = Ops<T>;
    uint32_t fa[4], fb[4];
    O::codes(wa, fa);
    O::codes(wb, fb);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        if (first) O::mma0(part[j], fa[0], fb[0], fa[1], fb[1], x[j].x, x[j].y);
        else O::mma(part[j], fa[0], fb[0], fa[1], fb[1], x[j].x, x[j].y);
        O::mma(part[j], fa[2], fb[2], fa[3], fb[3], x[j].z, x[j].w);
    }
}
template <int NT>
__device__ __forceinline__ void zero(float (&v)[NT][4]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
}
template <int NT>
__device__ __forceinline__ void add_scaled(float (&acc)[NT][4], const float (&part)[NT][4], float sa, float sb) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        acc[j][0] = fmaf(sa, part[j][0], acc[j][0]);
        acc[j][1] = fmaf(sa, part[j][1], acc[j][1]);
        acc[j][2] = fmaf(sb, part[j][2], acc[j][2]);
        acc[j][3] = fmaf(sb, part[j][3], acc[j][3]);
    }
}
// This lane's part of the 16-channel tile at rows [0, 16) of dst, row stride kRow.
template <int NT>
__device__ __forceinline__ void put_acc(float* dst, int kRow, const float (&acc)[NT][4], int g, int t) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float* d = dst + g * kRow + j * 8 + 2 * t;
        d[0] = acc[j][0];
        d[1] = acc[j][1];
        d[8 * kRow] = acc[j][2];
        d[8 * kRow + 1] = acc[j][3];
    }
}

// ── few rows ────────────────────────────────────────────────────────────────
__host__ __device__ constexpr int few_smem(int NT, int MT) { return kWarps * 16 * MT * (NT * 8 + 1) * 4; }

// A scale as it lies in memory, and its value.
__device__ __forceinline__ uint32_t raw_scale(const void* s, bool f32, int64_t i) {
    return f32 ? static_cast<const uint32_t*>(s)[i] : static_cast<const uint16_t*>(s)[i];
}
__device__ __forceinline__ float scale_value(uint32_t raw, int dt) {
    if (dt == SFB_F16) return __half2float(__ushort_as_half(static_cast<unsigned short>(raw)));
    return __uint_as_float(dt == SFB_BF16 ? raw << 16 : raw);
}

template <typename T, int G, int NT, int MT>
__global__ void __launch_bounds__(kThreads) w4a16_few_kernel(const W4Params p, const int act) {
    constexpr int kB = block_of(G), kQ = kB / 32, kBlocks = kChunk / kB, kU = kChunk / G;
    extern __shared__ float red[];
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * (16 * MT), m0 = blockIdx.y * (NT * 8);
    const int whole = p.K / kChunk, chunks = (p.K + kChunk - 1) / kChunk;
    const uint8_t* wr[2 * MT];                     // channels g, g + 8 of each tile; past the last: not stored
    int64_t sr[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int64_t n = min(n0 + 8 * i + g, p.N - 1);
        wr[i] = p.w + n * (p.K / 2) + t * (kB / 8);
        sr[i] = n * p.groups;
    }
    const T* xrow[NT];
    bool xok[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int m = m0 + j * 8 + g;
        xok[j] = m < p.M;
        xrow[j] = static_cast<const T*>(p.x) + static_cast<int64_t>(xok[j] ? m : 0) * p.ldx + t * (kB / 4);
    }
    const bool f32 = p.scale_dtype == SFB_F32;
    pdl_wait();
    struct Set { uint32_t w[2 * MT][4]; uint4 x[4][NT]; uint32_t s[2 * MT][kU]; };
    // kTail: the chunk ends before 128 inputs; what is past K is zeros
    auto load = [&](Set& s, int c, auto tail) {
        constexpr bool kTail = decltype(tail)::value;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            const int k0 = c * kChunk + k * kB;
            const bool in = !kTail || k0 < p.K;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                if constexpr (kQ == 2) {
                    const uint2 v = in ? *reinterpret_cast<const uint2*>(wr[i] + k0 / 2) : make_uint2(0, 0);
                    s.w[i][2 * k] = v.x; s.w[i][2 * k + 1] = v.y;
                } else {
                    s.w[i][k] = in ? *reinterpret_cast<const uint32_t*>(wr[i] + k0 / 2) : 0u;
                }
            }
#pragma unroll
            for (int q = 0; q < kQ; ++q)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    s.x[k * kQ + q][j] = in && xok[j] ? *reinterpret_cast<const uint4*>(xrow[j] + k0 + q * 8) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
                s.s[i][u] = !kTail || c * kU + u < p.groups ? raw_scale(p.scale, f32, sr[i] + c * kU + u) : 0u;
    };
    auto fetch = [&](Set& s, int c) {
        if (c < whole) load(s, c, std::false_type());
        else if (c < chunks) load(s, c, std::true_type());
    };
    float acc[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) zero(acc[i]);
    auto work = [&](const Set& s) {
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float part[NT][4];
#pragma unroll
                for (int w = u * (4 / kU); w < (u + 1) * (4 / kU); ++w)
                    word_mma<T, NT>(part, s.w[2 * i][w], s.w[2 * i + 1][w], s.x[w], w == u * (4 / kU));
                add_scaled(acc[i], part, scale_value(s.s[2 * i][u], p.scale_dtype), scale_value(s.s[2 * i + 1][u], p.scale_dtype));
            }
    };
    Set a, b;
    int c = warp;
    fetch(a, c);
    while (c < chunks) {
        fetch(b, c + kWarps);
        work(a);
        c += kWarps;
        if (c >= chunks) break;
        fetch(a, c + kWarps);
        work(b);
        c += kWarps;
    }
    constexpr int kRow = NT * 8 + 1;
#pragma unroll
    for (int i = 0; i < MT; ++i) put_acc<NT>(red + (warp * MT + i) * 16 * kRow, kRow, acc[i], g, t);
    Epilogue<T, 16 * MT, NT * 8, kThreads, kWarps> e;
    e.before(p, n0, m0);
    __syncthreads();
    e.after(p, act, red);
}

// ── more rows ───────────────────────────────────────────────────────────────
// WM channel tiles of 16 by four parts of the inputs: a ring stage holds one chunk
// of X for each part.
constexpr int kParts = 4, kManyStages = 2;
constexpr int kManyPitch = kParts * kChunk * 2 + 16;             // bytes per row of X in a stage
__host__ __device__ constexpr int many_threads(int WM) { return kParts * WM * 32; }
__host__ __device__ constexpr int many_smem(int NT, int WM) {
    const int ring = kManyStages * NT * 8 * kManyPitch, red = kParts * WM * 16 * (NT * 8 + 1) * 4;
    return ring > red ? ring : red;
}

template <typename T, int G, int NT, int WM>
__global__ void __launch_bounds__(many_threads(WM)) w4a16_many_kernel(const W4Params p, const int act) {
    constexpr int kB = block_of(G), kQ = kB / 32, kBlocks = kChunk / kB, kU = kChunk / G;
    constexpr int WK = kParts, kStages = kManyStages, kPitch = kManyPitch, kRows = NT * 8;
    constexpr int kSpan = WK * kChunk;             // inputs of a stage
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int wm = warp % WM, wk = warp / WM;
    const int n0 = blockIdx.x * (16 * WM), m0 = blockIdx.y * kRows;
    const int steps = (p.K + kSpan - 1) / kSpan;
    const int64_t na = min(n0 + 16 * wm + g, p.N - 1), nb = min(n0 + 16 * wm + g + 8, p.N - 1);
    const uint8_t* wa = p.w + na * (p.K / 2) + t * (kB / 8);
    const uint8_t* wb = p.w + nb * (p.K / 2) + t * (kB / 8);
    const uint32_t sbase = ptx::smem_u32(smem);
    pdl_wait();
    auto copy = [&](int i) {                       // X of step i; zeros past M and K
        const int stage = i % kStages;
        for (int e = tid; e < kRows * (kSpan / 8); e += many_threads(WM)) {
            const int r = e / (kSpan / 8), c = e % (kSpan / 8), k = i * kSpan + c * 8;
            const bool in = m0 + r < p.M && k < p.K;
            const T* src = static_cast<const T*>(p.x) + (in ? static_cast<int64_t>(m0 + r) * p.ldx + k : 0);
            cp_async16(sbase + (stage * kRows + r) * kPitch + c * 16, src, in ? 16 : 0);
        }
    };
    struct Set { uint32_t a[4], b[4]; float sa[kU], sb[kU]; };
    auto load = [&](Set& s, int i) {
        const int c = i * WK + wk;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            const int k0 = c * kChunk + k * kB;
            const bool in = k0 < p.K;
            if constexpr (kQ == 2) {
                const uint2 x = in ? *reinterpret_cast<const uint2*>(wa + k0 / 2) : make_uint2(0, 0);
                const uint2 y = in ? *reinterpret_cast<const uint2*>(wb + k0 / 2) : make_uint2(0, 0);
                s.a[2 * k] = x.x; s.a[2 * k + 1] = x.y; s.b[2 * k] = y.x; s.b[2 * k + 1] = y.y;
            } else {
                s.a[k] = in ? *reinterpret_cast<const uint32_t*>(wa + k0 / 2) : 0u;
                s.b[k] = in ? *reinterpret_cast<const uint32_t*>(wb + k0 / 2) : 0u;
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int grp = c * kU + u;
            const bool in = grp < p.groups;
            s.sa[u] = in ? scale_at(p.scale, p.scale_dtype, na * p.groups + grp) : 0.f;
            s.sb[u] = in ? scale_at(p.scale, p.scale_dtype, nb * p.groups + grp) : 0.f;
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (i < steps) copy(i);
        cp_async_commit();
    }
    float acc[NT][4];
    zero(acc);
    Set cur, nxt;
    if (steps > 0) load(nxt, 0);
    for (int i = 0; i < steps; ++i) {
        cur = nxt;
        cp_async_wait<kStages - 2>();
        __syncthreads();                           // X of step i is there; step i − 1's stage is free
        if (i + kStages - 1 < steps) copy(i + kStages - 1);
        cp_async_commit();
        if (i + 1 < steps) load(nxt, i + 1);
        const uint8_t* xs = smem + (i % kStages) * kRows * kPitch + g * kPitch + wk * kChunk * 2 + t * (kB / 2);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float part[NT][4];
#pragma unroll
            for (int w = u * (4 / kU); w < (u + 1) * (4 / kU); ++w) {
                uint4 x[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    x[j] = *reinterpret_cast<const uint4*>(xs + j * 8 * kPitch + (w / kQ) * kB * 2 + (w % kQ) * 16);
                word_mma<T, NT>(part, cur.a[w], cur.b[w], x, w == u * (4 / kU));
            }
            add_scaled(acc, part, cur.sa[u], cur.sb[u]);
        }
    }
    Epilogue<T, 16 * WM, kRows, many_threads(WM), WK> e;
    e.before(p, n0, m0);
    cp_async_wait<0>();
    __syncthreads();                               // the ring becomes the joining buffer
    constexpr int kRow = kRows + 1;
    float* red = reinterpret_cast<float*>(smem);   // [WK][16·WM][kRow]
    put_acc<NT>(red + (wk * 16 * WM + 16 * wm) * kRow, kRow, acc, g, t);
    __syncthreads();
    e.after(p, act, red);
}

template <auto Kern>
int launch(int smem, int threads, int channels, int rows, const W4Params& p, int act, cudaStream_t s) {
    const int64_t bx = (static_cast<int64_t>(p.N) + channels - 1) / channels;
    static std::atomic<bool> done[64];             // kernel attributes, once per device (idempotent)
    std::atomic<bool>& set = done[device_info().ordinal & 63];
    if (!set.load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) { record_cuda_error(e, "w4a16 kernel attributes"); return SFB_ERR_CUDA; }
        prefer_max_shared(Kern);
        set.store(true, std::memory_order_release);
    }
    // a grid's y ends at 65535 row tiles: more rows are several launches
    const int64_t most = 65535ll * rows, ysz = p.y_f32 ? 4 : 2;
    for (int64_t m = 0; m < p.M; m += most) {
        W4Params q = p;
        q.M = static_cast<int32_t>(std::min<int64_t>(most, p.M - m));
        q.x = static_cast<const uint16_t*>(p.x) + m * p.ldx;
        q.y = static_cast<uint8_t*>(p.y) + m * p.ldy * ysz;
        if (p.residual != nullptr) q.residual = static_cast<const uint8_t*>(p.residual) + m * p.ldr * ysz;
        SFB_TRY(launch_kernel(Kern, dim3(static_cast<unsigned>(bx), static_cast<unsigned>((q.M + rows - 1) / rows)), threads,
                              smem, s, true, q, act));
    }
    return SFB_OK;
}

template <typename T, int G, int NT, int MT>
int few(const W4Params& p, int act, cudaStream_t s) {
    return launch<w4a16_few_kernel<T, G, NT, MT>>(few_smem(NT, MT), kThreads, 16 * MT, NT * 8, p, act, s);
}
template <typename T, int G, int NT, int WM>
int many(const W4Params& p, int act, cudaStream_t s) {
    return launch<w4a16_many_kernel<T, G, NT, WM>>(many_smem(NT, WM), many_threads(WM), 16 * WM, NT * 8, p, act, s);
}

template <typename T, int G>
int pick_nt(const W4Params& p, int act, cudaStream_t s) {
    if (p.M <= 16) {
        // 32 channels a CTA (X and the loop's arithmetic for two tiles) once those
        // are two CTAs for every SM: 8 and 16 rows of 16384 × 8192 29.0 and 46.7 µs,
        // with 16 channels 36.0 and 56.3
        const bool two = (p.N + 31) / 32 >= 2 * std::max(device_info().num_sms, 1);
        if (p.M <= 8) return two ? few<T, G, 1, 2>(p, act, s)
                                 : few<T, G, 1, 1>(p, act, s);
        return two ? few<T, G, 2, 2>(p, act, s)
                   : few<T, G, 2, 1>(p, act, s);
    }
    // 64 channels a CTA once those fill half the SMs. 67 rows, 2048 inputs, 64 and 32
    // channels a CTA: 4096 outputs 18.3 and 14.3 µs, 6144 20.9 and 27.0.
    const int64_t tiles = (static_cast<int64_t>(p.M) + 71) / 72;
    const bool wide = (p.N + 63) / 64 * tiles * 2 >= std::max(device_info().num_sms, 1);
    if (p.M <= 32) return wide ? many<T, G, 4, 4>(p, act, s)
                               : many<T, G, 4, 2>(p, act, s);
    return wide ? many<T, G, 9, 4>(p, act, s)
                : many<T, G, 9, 2>(p, act, s);
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
    // (the kernels' 32-bit indexes go up to a tile of channels or 512 inputs past the last)
    if (M < 0 || N <= 0 || K <= 0 || N > 0x7ffffc00 || K > 0x7ffffc00) return SFB_ERR_SHAPE;
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
