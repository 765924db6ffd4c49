// kv4_attn.cu — attention over the 4-bit K/V cache (sfb_kv4_attention).
//
//   out[r, :] = softmax_j( scale · q[r, :]·k[j, :] ) · v[j, :],  k, v = c·s
//
// The rows r of one K/V head are its queries: seq_q times the query heads that
// share it. The products run with the keys on the MMA's M side (mma.sync
// m16n8k16, fp16 operands, fp32 sums):
//   Sᵀ[16 keys, 8 rows] = K[16, D] · Qᵀ          A = K, straight from the codes
//   Oᵀ[D, 8 rows]      += Vᵀ[D, 16] · Pᵀ         A = Vᵀ, straight from the codes
// so that one to eight rows (a generated token, with or without grouped heads)
// fill the N = 8 side, and nothing but codes and scales is loaded: a warp
// turns them into MMA fragments in registers. The order of the contraction
// index is free as long as both operands use the same, which is what makes the
// loads whole: lane (g, t) = (lane / 4, lane % 4) holds for Sᵀ the channels
// [D/4·t, D/4·(t+1)) of keys g and g + 8 and for Oᵀ the channels [D/8·g,
// D/8·(g+1)) of keys 2t, 2t+1, 2t+8, 2t+9.
// A nibble becomes fp16 exactly with one bit operation and one add or fma
// (0x6400 | n = 1024 + n), the scale is one exact fp16 product (kv4.cu).
// Pᵀ moves from the accumulator's layout to the B operand's by two movmatrix.
//
// Softmax in base 2: the running reference of a row is raised only when a
// logit passes it by more than 8, so that P <= 256 fits fp16 and the rescaling
// of Oᵀ is rare; row sums are fp32 from the unrounded probabilities.
//
// Work split: a CTA takes a range of 16-key tiles of one (session, K/V head,
// row tile), its warps interleaved; partial (m, l, O) are joined in shared
// memory, and across a cluster of up to 16 CTAs through distributed shared
// memory: no workspace, no atomics, an order that does not change.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sfb {

struct Kv4AttnParams {
    Kv4Params c;
    const void* q;
    void* out;
    int64_t q_st[3], o_st[3];
    int32_t H, g, Sq, Sk, R;          // g = H / Hkv query heads per K/V head, R = Sq · g rows
    int32_t rtiles, splits, causal;
    float sl2;                        // scale · log2(e)
    const int32_t* kv_len;
    const uint8_t* key_mask;
    int64_t mask_sb;
};

namespace kv4tc { template <typename T> int pick(Kv4AttnParams& p, int num_splits, cudaStream_t s); }

namespace kv4 {

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
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

template <int D> struct KWords;
template <> struct KWords<64>  { using T = uint2; };
template <> struct KWords<128> { using T = uint4; };
template <int D> struct VWords;
template <> struct VWords<64>  { using T = uint32_t; };
template <> struct VWords<128> { using T = uint2; };

// Codes and scales of one 16-key tile as a lane holds them.
template <int D>
struct Raw {
    typename KWords<D>::T k[2];       // keys g, g + 8: channels [D/4·t, +D/4)
    typename VWords<D>::T v[4];       // keys 2t, 2t+1, 2t+8, 2t+9: channels [D/8·g, +D/8)
    uint16_t ks[2], vs[4];
};

__host__ __device__ constexpr int attn_pad(int D) { return D + 8; }                  // halves per row of Q in shared memory
__host__ __device__ constexpr int attn_smem(int D, int NT, int W) {
    const int rows = NT * 8;
    return rows * attn_pad(D) * 2                                // Q
         + W * rows * D * 4 + W * rows * 2 * 4                   // per-warp O, m, l
         + rows * D * 4 + rows * 2 * 4;                          // the CTA's partial
}

template <typename T, int D, int NT, int W>
__global__ void __launch_bounds__(W * 32, NT == 1 ? 2 : 1) kv4_attn_kernel(const Kv4AttnParams p) {
    constexpr int kRows = NT * 8, kPad = attn_pad(D), kSteps = D / 16, kMT = D / 16;
    extern __shared__ __align__(16) uint8_t smem[];
    __half* sQ = reinterpret_cast<__half*>(smem);
    float* sO = reinterpret_cast<float*>(smem + kRows * kPad * 2);        // [W][kRows][D]
    float* sM = sO + W * kRows * D;                                       // [W][kRows]
    float* sL = sM + W * kRows;
    float* pO = sL + W * kRows;                                           // [kRows][D]
    float* pM = pO + kRows * D;
    float* pL = pM + kRows;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y / p.rtiles, rt = blockIdx.y - hk * p.rtiles, b = blockIdx.z;
    const int r0 = rt * kRows, rows = min(kRows, p.R - r0);
    pdl_trigger();
    pdl_wait();

    int n = p.Sk;                                                         // valid slots
    if (p.kv_len != nullptr) n = min(n, max(0, p.kv_len[b]));
    // a row sees the slots below limit(row)
    auto limit = [&](int r) { return p.causal ? min(n, max(0, n - p.Sq + r / p.g + 1)) : n; };
    const int kend = limit(r0 + rows - 1), kfull = limit(r0);             // limits grow with the row
    const int tiles = (kend + 15) >> 4;
    const int per = tiles / p.splits, rem = tiles - per * p.splits;
    const int t_begin = split * per + min(split, rem), t_end = t_begin + per + (split < rem ? 1 : 0);

    // ── Q rows as fp16 in shared memory (zeros past the last row) ───────────
    bool bad = false;
    for (int i = tid; i < kRows * (D / 8); i += W * 32) {
        const int r = i / (D / 8), d = (i % (D / 8)) * 8;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const int rr = r0 + r, qi = rr / p.g, h = hk * p.g + (rr - qi * p.g);
            const T* src = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + qi * p.q_st[2] + d;
            u = *reinterpret_cast<const uint4*>(src);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = __uint_as_float(w[e] << 16), hi = __uint_as_float(w[e] & 0xffff0000u);
                    bad |= (fabsf(lo) > 65504.f && !isinf(lo)) | (fabsf(hi) > 65504.f && !isinf(hi));
                    w[e] = h2u(__floats2half2_rn(lo, hi));
                }
            }
        }
        *reinterpret_cast<uint4*>(sQ + r * kPad + d) = u;
    }
    __syncthreads();

    const uint8_t* mask = p.key_mask != nullptr ? p.key_mask + b * p.mask_sb : nullptr;
    auto seen = [&](int key) { return key < kend && (mask == nullptr || mask[key] != 0); };
    // this lane's codes and scales of tile `warp` of the CTA, advanced by W tiles
    const int64_t first = static_cast<int64_t>(t_begin + warp) * 16;
    const uint8_t* kp = p.c.kc + b * p.c.code_sb + hk * p.c.code_sh + (first + g) * (D / 2) + (D / 8) * t;
    const uint8_t* vp = p.c.vc + b * p.c.code_sb + hk * p.c.code_sh + (first + 2 * t) * (D / 2) + (D / 16) * g;
    const uint16_t* ksp = reinterpret_cast<const uint16_t*>(p.c.ks + b * p.c.sc_sb + hk * p.c.sc_sh) +
                          (first + g) * (D / kGroup) + (D / 4 * t) / kGroup;
    const uint16_t* vsp = reinterpret_cast<const uint16_t*>(p.c.vs + b * p.c.sc_sb + hk * p.c.sc_sh) +
                          (first + 2 * t) * (D / kGroup) + (D / 8 * g) / kGroup;
    // In a tile with slots that are not seen, those are not read (nor trusted:
    // they may hold anything) and their scale is 0.
    auto load = [&](Raw<D>& r, int tile) {
        const int k0 = tile * 16;
        using KT = typename KWords<D>::T;
        using VT = typename VWords<D>::T;
        if (k0 + 16 <= kend && mask == nullptr) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                r.k[i] = *reinterpret_cast<const KT*>(kp + 8 * i * (D / 2));
                r.ks[i] = ksp[8 * i * (D / kGroup)];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (i & 1) + 8 * (i >> 1);
                r.v[i] = *reinterpret_cast<const VT*>(vp + row * (D / 2));
                r.vs[i] = vsp[row * (D / kGroup)];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                r.k[i] = {}; r.ks[i] = 0;
                if (k0 + g + 8 * i < kend) {
                    r.k[i] = *reinterpret_cast<const KT*>(kp + 8 * i * (D / 2));
                    r.ks[i] = ksp[8 * i * (D / kGroup)];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (i & 1) + 8 * (i >> 1);
                r.v[i] = {}; r.vs[i] = 0;
                if (seen(k0 + 2 * t + row)) {
                    r.v[i] = *reinterpret_cast<const VT*>(vp + row * (D / 2));
                    r.vs[i] = vsp[row * (D / kGroup)];
                }
            }
        }
        kp += 16 * W * (D / 2); vp += 16 * W * (D / 2);
        ksp += 16 * W * (D / kGroup); vsp += 16 * W * (D / kGroup);
    };

    float o[kMT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        m[j][0] = m[j][1] = -INFINITY;
        l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int i = 0; i < kMT; ++i) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    }
    constexpr bool kQReg = NT <= 2;                // Q fragments held in registers
    uint4 qr[kQReg ? NT : 1][kQReg ? kSteps / 2 : 1];
    if constexpr (kQReg) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int s = 0; s < kSteps / 2; ++s)
                qr[j][s] = reinterpret_cast<const uint4*>(sQ + (j * 8 + g) * kPad + (D / 4) * t)[s];
    }
    auto step = [&](const Raw<D>& cur, int tile) {
        const int k0 = tile * 16;
        // K fragments: half2 2s and 2s+1 of a key's words are step s
        uint32_t ka[2][kSteps * 2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&cur.k[i]);
            const __half2 s = __half2half2(__ushort_as_half(cur.ks[i]));
#pragma unroll
            for (int x = 0; x < kSteps / 2; ++x) {
                uint32_t d4[4];
                dequant_word(w[x], s, d4);
#pragma unroll
                for (int e = 0; e < 4; ++e) ka[i][4 * x + e] = d4[e];
            }
        }
        // Vᵀ fragments: words of a key pair interleaved by halves, so that a
        // nibble pair is one channel of both keys; [pair][word][low / high half]
        uint32_t va[2][kMT / 4][2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&cur.v[2 * i]);
            const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&cur.v[2 * i + 1]);
            const __half2 s = __halves2half2(__ushort_as_half(cur.vs[2 * i]), __ushort_as_half(cur.vs[2 * i + 1]));
#pragma unroll
            for (int x = 0; x < kMT / 4; ++x) {
                dequant_word(ptx::prmt(w0[x], w1[x], 0x5410u), s, va[i][x][0]);
                dequant_word(ptx::prmt(w0[x], w1[x], 0x7632u), s, va[i][x][1]);
            }
        }
        const bool edge = k0 + 16 > kfull || mask != nullptr;
        bool vis0 = true, vis1 = true;
        if (edge) { vis0 = seen(k0 + g); vis1 = seen(k0 + g + 8); }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float c[4] = {0.f, 0.f, 0.f, 0.f}, c2[4] = {0.f, 0.f, 0.f, 0.f};      // two chains
#pragma unroll
            for (int s = 0; s < kSteps; s += 2) {
                uint4 q4;
                if constexpr (kQReg) q4 = qr[j][s / 2];
                else q4 = reinterpret_cast<const uint4*>(sQ + (j * 8 + g) * kPad + (D / 4) * t)[s / 2];
                mma16816(c, ka[0][2 * s], ka[1][2 * s], ka[0][2 * s + 1], ka[1][2 * s + 1], q4.x, q4.y);
                mma16816(c2, ka[0][2 * s + 2], ka[1][2 * s + 2], ka[0][2 * s + 3], ka[1][2 * s + 3], q4.z, q4.w);
            }
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (c[e] + c2[e]) * p.sl2;
            if (edge) {
                const int ra = min(r0 + j * 8 + 2 * t, p.R - 1), rb = min(r0 + j * 8 + 2 * t + 1, p.R - 1);
                const int la = limit(ra), lb = limit(rb);
                if (!vis0 || k0 + g >= la) x[0] = -INFINITY;
                if (!vis0 || k0 + g >= lb) x[1] = -INFINITY;
                if (!vis1 || k0 + g + 8 >= la) x[2] = -INFINITY;
                if (!vis1 || k0 + g + 8 >= lb) x[3] = -INFINITY;
            }
            float ma = fmaxf(x[0], x[2]), mb = fmaxf(x[1], x[3]);
            if (__any_sync(0xffffffffu, ma > m[j][0] + 8.f || mb > m[j][1] + 8.f)) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, off));
                    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, off));
                }
                float aa = 1.f, ab = 1.f;
                if (ma > m[j][0] + 8.f) { aa = m[j][0] == -INFINITY ? 0.f : ptx::ex2(m[j][0] - ma); m[j][0] = ma; }
                if (mb > m[j][1] + 8.f) { ab = m[j][1] == -INFINITY ? 0.f : ptx::ex2(m[j][1] - mb); m[j][1] = mb; }
                l[j][0] *= aa; l[j][1] *= ab;
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                    o[i][j][0] *= aa; o[i][j][1] *= ab; o[i][j][2] *= aa; o[i][j][3] *= ab;
                }
            }
            const float ua = m[j][0] == -INFINITY ? 0.f : m[j][0], ub = m[j][1] == -INFINITY ? 0.f : m[j][1];
            const float p0 = ptx::ex2(x[0] - ua), p1 = ptx::ex2(x[1] - ub);
            const float p2 = ptx::ex2(x[2] - ua), p3 = ptx::ex2(x[3] - ub);
            l[j][0] += p0 + p2;
            l[j][1] += p1 + p3;
            const uint32_t b0 = movmatrix_t(h2u(__floats2half2_rn(p0, p1)));
            const uint32_t b1 = movmatrix_t(h2u(__floats2half2_rn(p2, p3)));
#pragma unroll
            for (int i = 0; i < kMT; ++i)
                mma16816(o[i][j], va[0][i / 4][0][i % 4], va[0][i / 4][1][i % 4], va[1][i / 4][0][i % 4],
                         va[1][i / 4][1][i % 4], b0, b1);
        }
    };
    // tiles in flight per warp: two where the registers allow two CTAs per SM all the same
    constexpr int kDepth = (NT == 1 && D == 64) ? 2 : 1;
    Raw<D> ring[kDepth];
    int tile = t_begin + warp;
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (tile + i * W < t_end) load(ring[i], tile + i * W);
    for (; tile < t_end; tile += kDepth * W) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            const int cur_tile = tile + i * W;
            if (i > 0 && cur_tile >= t_end) break;
            const Raw<D> cur = ring[i];
            if (cur_tile + kDepth * W < t_end) load(ring[i], cur_tile + kDepth * W);
            step(cur, cur_tile);
        }
    }

    // ── join the warps ──────────────────────────────────────────────────────
    // a lane holds, of rows 8j + 2t and + 1, the channels [D/8·g, +D/8): value
    // 8x + 2y + e of them is o[4x + y][j][row + 2e]
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float ls = l[j][e];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
            const int r = j * 8 + 2 * t + e;
            if (g == 0) { sM[warp * kRows + r] = m[j][e]; sL[warp * kRows + r] = ls; }
            float* dst = sO + (warp * kRows + r) * D + (D / 8) * g;
#pragma unroll
            for (int x = 0; x < kMT / 2; ++x)
                *reinterpret_cast<float4*>(dst + 4 * x) =
                    make_float4(o[2 * x][j][e], o[2 * x][j][e + 2], o[2 * x + 1][j][e], o[2 * x + 1][j][e + 2]);
        }
    }
    __syncthreads();
    T* out = static_cast<T*>(p.out);
    auto store = [&](int r, int d, float4 a, float inv) {
        const int rr = r0 + r, qi = rr / p.g, h = hk * p.g + (rr - qi * p.g);
        T* dst = out + b * p.o_st[0] + h * p.o_st[1] + qi * p.o_st[2] + d;
        uint2 u;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
            u.x = *reinterpret_cast<const uint32_t*>(&x); u.y = *reinterpret_cast<const uint32_t*>(&y);
        } else {
            u.x = h2u(__floats2half2_rn(a.x * inv, a.y * inv)); u.y = h2u(__floats2half2_rn(a.z * inv, a.w * inv));
        }
        *reinterpret_cast<uint2*>(dst) = u;
    };
    for (int i = tid; i < rows * (D / 4); i += W * 32) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        float M = -INFINITY, L = 0.f;
        for (int w = 0; w < W; ++w) M = fmaxf(M, sM[w * kRows + r]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; ++w) {
            const float mw = sM[w * kRows + r], lw = sL[w * kRows + r];
            if (mw == -INFINITY) { L += lw; continue; }       // 0, or NaN where every logit was
            const float f = ptx::ex2(mw - M);
            L += f * lw;
            const float4 v = *reinterpret_cast<const float4*>(sO + (w * kRows + r) * D + d);
            a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
        }
        if (p.splits == 1) {
            store(r, d, a, L != 0.f ? 1.f / L : 0.f);
        } else {
            *reinterpret_cast<float4*>(pO + r * D + d) = a;
            if (d == 0) { pM[r] = M; pL[r] = L; }
        }
    }
    if (p.splits > 1) {
        // ── join the cluster: CTA `split` finishes every splits-th row ──────
        ptx::cluster_sync();                       // every partial is written
        const uint32_t aO = ptx::smem_u32(pO), aM = ptx::smem_u32(pM), aL = ptx::smem_u32(pL);
        const int mine = split < rows ? (rows - split + p.splits - 1) / p.splits : 0;
        for (int i = tid; i < mine * (D / 4); i += W * 32) {
            const int r = split + (i / (D / 4)) * p.splits, d = (i % (D / 4)) * 4;
            float M = -INFINITY, L = 0.f;
            for (int k = 0; k < p.splits; ++k) M = fmaxf(M, ptx::dsmem_ld_f32(ptx::dsmem_map(aM + 4 * r, k)));
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < p.splits; ++k) {
                const float mk = ptx::dsmem_ld_f32(ptx::dsmem_map(aM + 4 * r, k));
                const float lk = ptx::dsmem_ld_f32(ptx::dsmem_map(aL + 4 * r, k));
                if (mk == -INFINITY) { L += lk; continue; }
                const float f = ptx::ex2(mk - M);
                L += f * lk;
                const float4 v = ptx::dsmem_ld_f32x4(ptx::dsmem_map(aO + 4 * (r * D + d), k));
                a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
            }
            store(r, d, a, L != 0.f ? 1.f / L : 0.f);
        }
        ptx::cluster_sync();                       // nobody leaves while its partial may be read
    }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
}

template <typename T, int D, int NT, int W>
int launch_attn(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    const DeviceInfo& dev = device_info();
    constexpr int smem = attn_smem(D, NT, W);
    static_assert(smem <= 227 * 1024, "shared memory budget");
    auto kern = kv4_attn_kernel<T, D, NT, W>;
    static std::atomic<bool> done[64];             // kernel attributes, once per device (idempotent)
    if (!done[dev.ordinal & 63].load(std::memory_order_acquire)) {
        const cudaError_t e1 = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        const cudaError_t e2 = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e1 != cudaSuccess || e2 != cudaSuccess) {
            record_cuda_error(e1 != cudaSuccess ? e1 : e2, "kv4 attention attributes");
            return SFB_ERR_CUDA;
        }
        prefer_max_shared(kern);
        done[dev.ordinal & 63].store(true, std::memory_order_release);
    }
    p.rtiles = (p.R + NT * 8 - 1) / (NT * 8);
    const int64_t units = static_cast<int64_t>(p.c.B) * p.c.Hkv * p.rtiles;
    const int tiles = (p.Sk + 15) / 16;
    int sp = num_splits;
    if (sp == 0) {
        // enough CTAs for every SM, at least two tiles for each of a CTA's warps
        sp = static_cast<int>(std::min<int64_t>(16, std::max<int64_t>(1, dev.num_sms / units)));
        sp = std::min(sp, std::max(1, tiles / (2 * W)));
    }
    p.splits = std::min(sp, std::max(1, tiles));
    if (static_cast<int64_t>(p.c.Hkv) * p.rtiles > 65535 || p.c.B > 65535) return SFB_ERR_SHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.c.Hkv * p.rtiles, p.c.B);
    cfg.blockDim = dim3(W * 32, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + pdl_attr(&attr[1], true);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) { record_cuda_error(e, "kv4 attention launch"); return SFB_ERR_LAUNCH; }
    return SFB_OK;
}

template <typename T>
int pick_attn(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    if (p.c.D == 64) {
        if (p.R <= 8) return launch_attn<T, 64, 1, 8>(p, num_splits, s);
        if (p.R <= 16) return launch_attn<T, 64, 2, 8>(p, num_splits, s);
        return kv4tc::pick<T>(p, num_splits, s);
    }
    if (p.R <= 8) return launch_attn<T, 128, 1, 8>(p, num_splits, s);
    if (p.R <= 16) return launch_attn<T, 128, 2, 8>(p, num_splits, s);
    return launch_attn<T, 128, 4, 8>(p, num_splits, s);
}

}  // namespace kv4

int kv4_attention_launch(const sfb_kv4_cache* cache, const sfb_kv4_attn_args& a, cudaStream_t s) {
    Kv4AttnParams p{};
    SFB_TRY(kv4_cache_check(cache, p.c));
    if (a.dtype != SFB_F16 && a.dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (a.heads < 1 || a.heads % p.c.Hkv != 0 || a.seq_q < 0 || a.seq_k < 0 || a.seq_k > p.c.cap) return SFB_ERR_SHAPE;
    if (a.num_splits < 0 || a.num_splits > 16) return SFB_ERR_INVALID;
    if (p.c.B == 0 || a.seq_q == 0) return SFB_OK;
    if (a.q == nullptr || a.out == nullptr) return SFB_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15u) return SFB_ERR_ALIGN;
    for (int i = 0; i < 3; ++i)
        if (a.q_stride[i] % 8 || a.out_stride[i] % 8) return SFB_ERR_ALIGN;
    const int64_t R = static_cast<int64_t>(a.seq_q) * (a.heads / p.c.Hkv);
    if (R > 0x7fffff00) return SFB_ERR_SHAPE;
    if (!is_sm100(device_info())) return SFB_ERR_UNSUPPORTED;
    p.q = a.q; p.out = a.out;
    for (int i = 0; i < 3; ++i) { p.q_st[i] = a.q_stride[i]; p.o_st[i] = a.out_stride[i]; }
    p.H = a.heads; p.g = a.heads / p.c.Hkv; p.Sq = a.seq_q; p.Sk = a.seq_k; p.R = static_cast<int32_t>(R);
    p.causal = a.is_causal ? 1 : 0;
    p.sl2 = (a.scale == 0.f ? 1.f / sqrtf(static_cast<float>(p.c.D)) : a.scale) * 1.4426950408889634f;
    p.kv_len = a.kv_len; p.key_mask = a.key_mask; p.mask_sb = a.key_mask_stride_b;
    if (a.dtype == SFB_BF16) return kv4::pick_attn<__nv_bfloat16>(p, a.num_splits, s);
    return kv4::pick_attn<__half>(p, a.num_splits, s);
}

}  // namespace sfb
