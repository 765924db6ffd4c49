// kv4_attn.cu — attention over the 4-bit K/V cache (sfb_kv4_attention), up to 8
// rows per K/V head; kv4_attn_tc.cu has the form for more.
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
// [D/4·t, D/4·(t+1)) of the keys of MMA rows g and g + 8 and for Oᵀ the channels
// [D/8·g, D/8·(g+1)) of rows 2t, 2t+1, 2t+8, 2t+9. Row m of the MMA is key
// key_of(m) of its tile, chosen so that either kind of load touches one
// contiguous run of shared memory.
// A tile is 16 keys; blocks of 128 give one to each of a CTA's eight warps. With
// 64 channels a lane loads its codes straight into registers, two tiles ahead of
// the one it works on. With 128 those registers would cost the second CTA
// per SM, so blocks go through a ring in shared memory, four untiled bulk copies
// each (codes and scales of K and V), issued by a ninth warp. 32 sessions of 8 to
// 16 k slots of 8 heads: 178 µs from registers, 153 through the ring (144 as it is
// now: 3.2 TB/s of codes and scales); 32 sessions of 4374 slots of 32 64-channel
// heads: 105 µs from registers (101 now, 3.2 TB/s), 111 through the ring; one session
// of those 7.9 µs, 1.5 of them the launch. (Device times, calls back to back from a
// graph; an eager call costs the host 11 µs.) What bounds both is the issue of
// instructions, most of them to make fragments of the codes, together with the
// dependence of a tile's steps on one another: with 128 channels 400 instructions a
// tile and warp are 56 % of the issue slots, at 24 % of an SM's warps.
// A nibble becomes fp16 exactly with one bit operation and one add or fma
// (0x6400 | n = 1024 + n), the scale is one exact fp16 product (kv4.cu).
// Pᵀ moves from the accumulator's layout to the B operand's by two movmatrix.
//
// Softmax in base 2, P = exp2(x − m) against a row's running reference m, rounded to
// fp16 for the tensor cores (half a step is 2^-11 of it: lost beside a bf16 result's
// rounding, not beside an fp16 one's). m is put 7 below the largest logit and raised
// only when one passes it by more than 15: rescaling Oᵀ is rare, P <= 2^15 fits, and a
// probability keeps all of its bits down to 2^-21 of the row's largest, some down to
// 2^-31. (With m at the largest that ended at 2^-14 and 2^-24, and a row whose largest
// probability had a V near 0 lost the result of the others.) Row sums are fp32 from the
// unrounded probabilities.
//
// Work split: a CTA takes a range of the 128-key blocks of one (session, K/V head),
// a 16-key tile of each block to a warp; partial (m, l, O) are joined in shared
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
    int32_t g, Sq, Sk, R;             // g query heads per K/V head, R = Sq · g rows
    int32_t rtiles, splits, causal;
    int32_t rt0, ytiles;              // of a launch: first row tile, row tiles
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
template <int D> struct KWords;
template <> struct KWords<64>  { using T = uint2; };
template <> struct KWords<128> { using T = uint4; };
template <int D> struct VWords;
template <> struct VWords<64>  { using T = uint32_t; };
template <> struct VWords<128> { using T = uint2; };

// A scale that is not finite makes its group NaN. For a slot that only some of a
// tile's rows see (causal calls) the others would take 0 · NaN from such a V, so
// there V is taken as 0 and K as NaN: the rows that see the slot become NaN whole.
__device__ __forceinline__ bool not_finite(uint32_t scale_bits) { return (scale_bits & 0x7c00u) == 0x7c00u; }
__device__ __forceinline__ void contain(__half2& ks, __half2& vs) {
    const uint32_t v = h2u(vs);
    if (not_finite(v) || not_finite(v >> 16)) { ks = u2h(0x7fff7fffu); vs = u2h(0u); }
}

// A query's infinity as NaN: it makes every logit of its row an infinity or NaN, and
// so the row NaN, but logits that are minus infinity throughout would pass for masked.
__device__ __forceinline__ uint32_t inf_to_nan(uint32_t q2) {
    const __half2 q = u2h(q2);
    return h2u(__hadd2(q, __hsub2(q, q)));
}

constexpr float kUnseen = 1e30f;
// A row's reference is put kBelow under its largest logit, and raised when one passes it by more than kOver.
constexpr float kBelow = 7.f, kOver = 15.f;
constexpr int kRows = 8;                                         // rows of a CTA
constexpr int kWarps = 8;                                        // computing
__host__ __device__ constexpr bool uses_ring(int D) { return D == 128; }
__host__ __device__ constexpr int attn_threads(int D) { return (kWarps + (uses_ring(D) ? 1 : 0)) * 32; }   // a ninth warp issues the copies
constexpr int kBlock = 16 * kWarps;                              // keys per ring stage
__host__ __device__ constexpr int code_bytes(int D) { return kBlock * D / 2; }
__host__ __device__ constexpr int scale_bytes(int D) { return kBlock * (D / kGroup) * 2; }
__host__ __device__ constexpr int stage_bytes(int D) { return 2 * (code_bytes(D) + scale_bytes(D)); }
__host__ __device__ constexpr int ring_stages(int D) { return uses_ring(D) ? 4 : 0; }
__host__ __device__ constexpr int attn_pad(int D) { return D + 8; }   // halves per row of Q in shared memory
__host__ __device__ constexpr int join_bytes(int D) {         // per-warp O, m, l and the CTA's partial
    return (kWarps + 1) * kRows * (D + 2) * 4;
}
__host__ __device__ constexpr int attn_smem(int D) {
    const int ring = stage_bytes(D) * ring_stages(D), join = join_bytes(D);
    return kRows * attn_pad(D) * 2 + (ring > join ? ring : join) + 16 * ring_stages(D);
}
// Codes and scales of one 16-key tile as a lane holds them: K of MMA rows g and
// g + 8 (channels [D/4·t, +D/4)), V of rows 2t, 2t+1, 2t+8, 2t+9 (channels [D/8·g, +D/8)).
template <int D>
struct Raw {
    typename KWords<D>::T k[2];
    typename VWords<D>::T v[4];
    uint16_t ks[2], vs[4];
};

// The key of a 16-key tile that is row m of the MMAs.
__device__ __forceinline__ int key_of(int m) { return ((m & 7) >> 1) + 4 * (m & 1) + 8 * (m >> 3); }

template <typename T, int D>
__global__ void __launch_bounds__(attn_threads(D), 2) kv4_attn_kernel(const Kv4AttnParams p) {
    constexpr int kPad = attn_pad(D), kSteps = D / 16, kMT = D / 16, W = kWarps, kThreads = attn_threads(D);
    constexpr int kStages = ring_stages(D), kCode = code_bytes(D), kScale = scale_bytes(D), kStage = stage_bytes(D);
    extern __shared__ __align__(16) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem);                   // full, then empty
    __half* sQ = reinterpret_cast<__half*>(smem + 16 * kStages);
    uint8_t* ring = smem + 16 * kStages + kRows * kPad * 2;               // per stage: K codes, V codes, K, V scales
    float* sO = reinterpret_cast<float*>(ring);                           // over the ring at the end: [W][kRows][D]
    float* sM = sO + W * kRows * D;                                       // [W][kRows]
    float* sL = sM + W * kRows;
    float* pO = sL + W * kRows;                                           // [kRows][D]
    float* pM = pO + kRows * D;
    float* pL = pM + kRows;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const int rows = p.R;
    if (kStages > 0 && tid == 0) {
        for (int i = 0; i < kStages; ++i) { ptx::mbar_init(&bars[i], 1); ptx::mbar_init(&bars[kStages + i], W); }
        ptx::fence_mbarrier_init();
    }
    pdl_trigger();
    pdl_wait();

    int n = p.Sk;                                                         // valid slots
    if (p.kv_len != nullptr) n = min(n, max(0, p.kv_len[b]));
    // a row sees the slots below limit(row)
    auto limit = [&](int r) { return p.causal ? min(n, max(0, n - p.Sq + r / p.g + 1)) : n; };
    const int kend = limit(rows - 1), kfull = limit(0);             // limits grow with the row
    const int blocks = (kend + kBlock - 1) / kBlock;
    const int per = blocks / p.splits, rem = blocks - per * p.splits;
    const int b_begin = split * per + min(split, rem), nblk = per + (split < rem ? 1 : 0);

    // ── Q rows as fp16 in shared memory (zeros past the last row) ───────────
    bool bad = false;
    for (int i = tid; i < kRows * (D / 8); i += kThreads) {
        const int r = i / (D / 8), d = (i % (D / 8)) * 8;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const int qi = r / p.g, h = hk * p.g + (r - qi * p.g);
            const T* src = static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] + qi * p.q_st[2] + d;
            u = *reinterpret_cast<const uint4*>(src);
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    const float lo = __uint_as_float(w[e] << 16), hi = __uint_as_float(w[e] & 0xffff0000u);
                    bad |= (fabsf(lo) > 65504.f && !isinf(lo)) | (fabsf(hi) > 65504.f && !isinf(hi));
                    w[e] = h2u(__floats2half2_rn(lo, hi));
                }
                w[e] = inf_to_nan(w[e]);
            }
        }
        *reinterpret_cast<uint4*>(sQ + r * kPad + d) = u;
    }
    __syncthreads();

    const uint8_t* mask = p.key_mask != nullptr ? p.key_mask + b * p.mask_sb : nullptr;
    auto row_bad = [](const uint16_t* vs) {         // a slot's scales of V
        bool x = false;
#pragma unroll
        for (int i = 0; i < D / kGroup; ++i) x |= not_finite(vs[i]);
        return x;
    };
    auto seen = [&](int key) { return key < kend && (mask == nullptr || mask[key] != 0); };
    bool ok = true;

    const float sgn = p.sl2 < 0.f ? -1.f : 1.f;    // a masked logit is −∞ after the scaling
    float o[kMT][4], nm[2] = {kUnseen, kUnseen}, l[2] = {0.f, 0.f};      // nm: −reference
#pragma unroll
    for (int i = 0; i < kMT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    uint4 qr[kSteps / 2];                          // Q fragments
#pragma unroll
    for (int s = 0; s < kSteps / 2; ++s) qr[s] = reinterpret_cast<const uint4*>(sQ + g * kPad + (D / 4) * t)[s];
    auto step = [&](const Raw<D>& r, int k0) {
        const bool edge = k0 + 16 > kfull || mask != nullptr;
        // K fragments: half2 2s and 2s+1 of a key's words are step s
        uint32_t ka[2][kSteps * 2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&r.k[i]);
            const __half2 s = __half2half2(__ushort_as_half(r.ks[i]));
#pragma unroll
            for (int x = 0; x < kSteps / 2; ++x) {
                uint32_t d4[4];
                dequant_word(w[x], s, d4);
#pragma unroll
                for (int e = 0; e < 4; ++e) ka[i][4 * x + e] = d4[e];
            }
        }
        uint32_t pb[2];                            // Pᵀ fragments
        {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < kSteps; s += 2) {
                const uint4 q4 = qr[s / 2];
                mma16816(c, ka[0][2 * s], ka[1][2 * s], ka[0][2 * s + 1], ka[1][2 * s + 1], q4.x, q4.y);
                mma16816(c, ka[0][2 * s + 2], ka[1][2 * s + 2], ka[0][2 * s + 3], ka[1][2 * s + 3], q4.z, q4.w);
            }
            if (edge) {
                const int ra = min(2 * t, p.R - 1), rb = min(2 * t + 1, p.R - 1);
                const int la = limit(ra), lb = limit(rb), ka_ = k0 + key_of(g), kb_ = ka_ + 8;
                const bool v0 = seen(ka_), v1 = seen(kb_);
                if (!v0 || ka_ >= la) c[0] = -INFINITY * sgn;
                if (!v0 || ka_ >= lb) c[1] = -INFINITY * sgn;
                if (!v1 || kb_ >= la) c[2] = -INFINITY * sgn;
                if (!v1 || kb_ >= lb) c[3] = -INFINITY * sgn;
            }
            // exponents against the rows' references; a row that saw no key yet has
            // the reference −kUnseen, so that its first key passes it
            float x[4] = {fmaf(c[0], p.sl2, nm[0]), fmaf(c[1], p.sl2, nm[1]), fmaf(c[2], p.sl2, nm[0]),
                          fmaf(c[3], p.sl2, nm[1])};
            if (__any_sync(0xffffffffu, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > kOver)) {
                float ma = fmaxf(c[0] * p.sl2, c[2] * p.sl2), mb = fmaxf(c[1] * p.sl2, c[3] * p.sl2);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, off));
                    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, off));
                }
                float aa = 1.f, ab = 1.f;
                if (ma + nm[0] > kOver) { aa = nm[0] == kUnseen ? 0.f : ptx::ex2(kBelow - ma - nm[0]); nm[0] = kBelow - ma; }
                if (mb + nm[1] > kOver) { ab = nm[1] == kUnseen ? 0.f : ptx::ex2(kBelow - mb - nm[1]); nm[1] = kBelow - mb; }
                l[0] *= aa; l[1] *= ab;
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                    o[i][0] *= aa; o[i][1] *= ab; o[i][2] *= aa; o[i][3] *= ab;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(c[e], p.sl2, nm[e & 1]);
            }
            const float p0 = ptx::ex2(x[0]), p1 = ptx::ex2(x[1]), p2 = ptx::ex2(x[2]), p3 = ptx::ex2(x[3]);
            l[0] += p0 + p2;
            l[1] += p1 + p3;
            pb[0] = movmatrix_t(h2u(__floats2half2_rn(p0, p1)));
            pb[1] = movmatrix_t(h2u(__floats2half2_rn(p2, p3)));
        }
        // Vᵀ fragments: words of a key pair interleaved by halves, so that a
        // nibble pair is one channel of both keys; [pair][word][low / high half]
        uint32_t va[2][kMT / 4][2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&r.v[2 * i]);
            const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&r.v[2 * i + 1]);
            const __half2 s = __halves2half2(__ushort_as_half(r.vs[2 * i]), __ushort_as_half(r.vs[2 * i + 1]));
#pragma unroll
            for (int x = 0; x < kMT / 4; ++x) {
                dequant_word(ptx::prmt(w0[x], w1[x], 0x5410u), s, va[i][x][0]);
                dequant_word(ptx::prmt(w0[x], w1[x], 0x7632u), s, va[i][x][1]);
            }
        }
#pragma unroll
        for (int i = 0; i < kMT; ++i)
            mma16816(o[i], va[0][i / 4][0][i % 4], va[0][i / 4][1][i % 4], va[1][i / 4][0][i % 4],
                     va[1][i / 4][1][i % 4], pb[0], pb[1]);
    };
    if constexpr (!uses_ring(D)) {
        // the next tile's codes are in flight while this one is worked on; slots
        // that are not seen are not read
        const int64_t first = static_cast<int64_t>(b_begin) * kBlock + warp * 16;
        const int64_t hb = b * p.c.code_sb + hk * p.c.code_sh, hs = b * p.c.sc_sb + hk * p.c.sc_sh;
        using KT = typename KWords<D>::T;
        using VT = typename VWords<D>::T;
        const uint8_t* kp = p.c.kc + hb + (first + key_of(g)) * (D / 2) + (D / 8) * t;
        const uint8_t* vp = p.c.vc + hb + (first + t) * (D / 2) + (D / 16) * g;
        const uint16_t* ksp = reinterpret_cast<const uint16_t*>(p.c.ks + hs) + (first + key_of(g)) * (D / kGroup) + (D / 4 * t) / kGroup;
        const uint16_t* vsp = reinterpret_cast<const uint16_t*>(p.c.vs + hs) + (first + t) * (D / kGroup) + (D / 8 * g) / kGroup;
        auto load = [&](Raw<D>& r, int k0) {       // tiles in order: the pointers move along
            const bool whole = k0 + 16 <= kfull && mask == nullptr;
            if (whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    r.k[e] = *reinterpret_cast<const KT*>(kp + 8 * e * (D / 2));
                    r.ks[e] = ksp[8 * e * (D / kGroup)];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    r.v[e] = *reinterpret_cast<const VT*>(vp + 4 * e * (D / 2));
                    r.vs[e] = vsp[4 * e * (D / kGroup)];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    r.k[e] = {}; r.ks[e] = 0;
                    if (seen(k0 + key_of(g) + 8 * e)) {
                        r.k[e] = *reinterpret_cast<const KT*>(kp + 8 * e * (D / 2));
                        r.ks[e] = ksp[8 * e * (D / kGroup)];
                        const int key = k0 + key_of(g) + 8 * e;
                        if (key >= kfull && row_bad(reinterpret_cast<const uint16_t*>(p.c.vs + hs) + static_cast<int64_t>(key) * (D / kGroup)))
                            r.ks[e] = 0x7fff;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    r.v[e] = {}; r.vs[e] = 0;
                    if (seen(k0 + t + 4 * e)) {
                        r.v[e] = *reinterpret_cast<const VT*>(vp + 4 * e * (D / 2));
                        r.vs[e] = vsp[4 * e * (D / kGroup)];
                        if (k0 + t + 4 * e >= kfull && not_finite(r.vs[e])) r.vs[e] = 0;
                    }
                }
            }
            kp += kBlock * (D / 2); vp += kBlock * (D / 2);
            ksp += kBlock * (D / kGroup); vsp += kBlock * (D / kGroup);
        };
        const int k_end = min(kend, (b_begin + nblk) * kBlock);
        int k0 = static_cast<int>(first);
        // two tiles ahead, in three sets of registers by turns (copies between them
        // were a twentieth of a tile's instructions)
        Raw<D> ra, rb, rc;
        auto turn = [&](const Raw<D>& now, Raw<D>& later) {
            if (k0 + 2 * kBlock < k_end) load(later, k0 + 2 * kBlock);
            step(now, k0);
            k0 += kBlock;
            return k0 < k_end;
        };
        if (k0 < k_end) load(ra, k0);
        if (k0 + kBlock < k_end) load(rb, k0 + kBlock);
        while (k0 < k_end) {
            if (!turn(ra, rc)) break;
            if (!turn(rb, ra)) break;
            turn(rc, rb);
        }
    } else {
        // this lane's codes and scales of a tile in shared memory. Slots that are not
        // seen may hold anything: their scale is taken as 0.
        auto fetch = [&](Raw<D>& r, const uint8_t* kc, const uint8_t* vc, const uint16_t* ks, const uint16_t* vs,
                         int in_block, int k0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = in_block + key_of(g) + 8 * i;
                r.k[i] = *reinterpret_cast<const typename KWords<D>::T*>(kc + key * (D / 2) + (D / 8) * t);
                r.ks[i] = ks[key * (D / kGroup) + (D / 4 * t) / kGroup];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = in_block + t + 4 * i;            // key_of(2t + (i & 1) + 8·(i >> 1))
                r.v[i] = *reinterpret_cast<const typename VWords<D>::T*>(vc + key * (D / 2) + (D / 16) * g);
                r.vs[i] = vs[key * (D / kGroup) + (D / 8 * g) / kGroup];
            }
            if (k0 + 16 > kfull || mask != nullptr) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = k0 + key_of(g) + 8 * i;
                    if (!seen(key)) r.ks[i] = 0;
                    else if (key >= kfull && row_bad(vs + (in_block + key - k0) * (D / kGroup))) r.ks[i] = 0x7fff;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = k0 + t + 4 * i;
                    if (!seen(key) || (key >= kfull && not_finite(r.vs[i]))) r.vs[i] = 0;
                }
            }
        };
        // ── copies of block i (one lane), once its stage is free ───────────────
        auto copy_block = [&](int i) {
            const int s = i % kStages;
            if (i >= kStages && !ptx::mbar_wait(&bars[kStages + s], ((i / kStages) - 1) & 1)) return false;
            const int64_t hb = b * p.c.code_sb + hk * p.c.code_sh, hs = b * p.c.sc_sb + hk * p.c.sc_sh;
            const int64_t key0 = static_cast<int64_t>(b_begin + i) * kBlock;
            // whole groups of four slots: the capacity is a multiple of 4
            const uint32_t n4 = static_cast<uint32_t>(min(static_cast<int64_t>(kBlock), (kend + 3) / 4 * 4 - key0));
            const uint32_t cb = n4 * (D / 2), sb = n4 * (D / kGroup) * 2;
            uint8_t* st = ring + s * kStage;
            ptx::mbar_arrive_expect_tx(&bars[s], 2 * (cb + sb));
            ptx::bulk_load(st, p.c.kc + hb + key0 * (D / 2), cb, &bars[s]);
            ptx::bulk_load(st + kCode, p.c.vc + hb + key0 * (D / 2), cb, &bars[s]);
            ptx::bulk_load(st + 2 * kCode, p.c.ks + hs + key0 * (D / kGroup), sb, &bars[s]);
            ptx::bulk_load(st + 2 * kCode + kScale, p.c.vs + hs + key0 * (D / kGroup), sb, &bars[s]);
            return true;
        };
        int issued = 0;                                // blocks copied, in the copying lane
        if (warp == W) {
            while (lane == 0 && ok && issued < nblk) {
                if (copy_block(issued)) ++issued;
                else ok = false;
            }
        } else {
            auto take = [&](Raw<D>& r, int i) {
                const int s = i % kStages;
                if (!ok || !ptx::mbar_wait(&bars[s], (i / kStages) & 1)) ok = false;
                ok = __all_sync(0xffffffffu, ok) != 0;
                const uint8_t* st = ring + s * kStage;
                if (ok)
                    fetch(r, st, st + kCode, reinterpret_cast<const uint16_t*>(st + 2 * kCode),
                          reinterpret_cast<const uint16_t*>(st + 2 * kCode + kScale), warp * 16,
                          (b_begin + i) * kBlock + warp * 16);
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&bars[kStages + s]);
            };
            auto work = [&](const Raw<D>& r, int i) {
                const int k0 = (b_begin + i) * kBlock + warp * 16;
                if (ok && k0 < kend) step(r, k0);
            };
            Raw<D> r{};
            for (int i = 0; i < nblk; ++i) {
                take(r, i);
                work(r, i);
            }
        }
        // nothing is in flight when the ring becomes the joining buffer
        if (lane == 0)
            for (int i = max(0, issued - kStages); i < issued; ++i)
                if (!ptx::mbar_wait(&bars[i % kStages], (i / kStages) & 1)) ok = false;
    }
    __syncthreads();

    // ── join the warps ──────────────────────────────────────────────────────
    // a lane holds, of rows 2t and 2t + 1, the channels [D/8·g, +D/8): value
    // 8x + 2y + e of them is o[4x + y][row + 2e]
    if (warp < W) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float ls = l[e];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
            const int r = 2 * t + e;
            if (g == 0) { sM[warp * kRows + r] = nm[e] == kUnseen ? -INFINITY : -nm[e]; sL[warp * kRows + r] = ls; }
            float* dst = sO + (warp * kRows + r) * D + (D / 8) * g;
#pragma unroll
            for (int x = 0; x < kMT / 2; ++x)
                *reinterpret_cast<float4*>(dst + 4 * x) =
                    make_float4(o[2 * x][e], o[2 * x][e + 2], o[2 * x + 1][e], o[2 * x + 1][e + 2]);
        }
    }
    __syncthreads();
    T* out = static_cast<T*>(p.out);
    auto store = [&](int r, int d, float4 a, float inv) {
        const int qi = r / p.g, h = hk * p.g + (r - qi * p.g);
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
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
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
            if (ok) store(r, d, a, L != 0.f ? 1.f / L : 0.f);
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
        for (int i = tid; i < mine * (D / 4); i += kThreads) {
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
            if (ok) store(r, d, a, L != 0.f ? 1.f / L : 0.f);
        }
        ptx::cluster_sync();                       // nobody leaves while its partial may be read
    }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
    if (!ok) atomicExch(&g_sfb_device_error, SFB_ERR_DEVICE_TIMEOUT);
}

// Launches `kern` on a grid of (splits, K/V heads × row tiles, sessions). A grid's y
// and z end at 65535: longer ones are cut into several launches, whose pointers and
// first row tile are moved along.
inline int launch_ranges(void (*kern)(Kv4AttnParams), cudaLaunchConfig_t& cfg, const Kv4AttnParams& all, const char* what) {
    constexpr int kMax = 65535;
    const int heads = std::max(1, kMax / all.rtiles), rows = std::min(kMax, all.rtiles);
    for (int64_t b = 0; b < all.c.B; b += kMax)
        for (int64_t h = 0; h < all.c.Hkv; h += heads)
            for (int64_t t = 0; t < all.rtiles; t += rows) {
                Kv4AttnParams p = all;
                const int64_t code = b * p.c.code_sb + h * p.c.code_sh, scale = b * p.c.sc_sb + h * p.c.sc_sh;
                p.c.kc += code; p.c.vc += code; p.c.ks += scale; p.c.vs += scale;
                p.q = static_cast<const uint16_t*>(p.q) + b * p.q_st[0] + h * p.g * p.q_st[1];
                p.out = static_cast<uint16_t*>(p.out) + b * p.o_st[0] + h * p.g * p.o_st[1];
                if (p.kv_len != nullptr) p.kv_len += b;
                if (p.key_mask != nullptr) p.key_mask += b * p.mask_sb;
                p.rt0 = static_cast<int32_t>(t);
                p.ytiles = static_cast<int32_t>(std::min<int64_t>(rows, p.rtiles - t));
                cfg.gridDim = dim3(p.splits, static_cast<unsigned>(std::min<int64_t>(heads, p.c.Hkv - h) * p.ytiles),
                                   static_cast<unsigned>(std::min<int64_t>(kMax, p.c.B - b)));
                const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
                if (e != cudaSuccess) { record_cuda_error(e, what); return SFB_ERR_LAUNCH; }
            }
    return SFB_OK;
}

template <typename T, int D>
int launch_attn(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    const DeviceInfo& dev = device_info();
    constexpr int smem = attn_smem(D);
    static_assert(smem <= 227 * 1024, "shared memory budget");
    auto kern = kv4_attn_kernel<T, D>;
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
    const int64_t units = static_cast<int64_t>(p.c.B) * p.c.Hkv;
    const int blocks = (p.Sk + kBlock - 1) / kBlock;
    int sp = num_splits;
    if (sp == 0) {
        // Two CTAs for every SM (a power of two: a cluster of 8 measured 43 µs
        // where 12 took 56, 4 sessions of 8 heads and 16 k slots). With more units
        // than that, cut the long ones into 4096 slots and more until there are
        // about 1024 CTAs, so that sessions of different lengths fill the SMs
        // evenly (32 of 8 to 16 k slots, 8 heads: 145 µs, 162 without). At least a
        // block a CTA.
        const int64_t fill = std::max<int64_t>(1, 2 * dev.num_sms / units);
        sp = 1;
        while (sp < 16 && 2 * sp <= fill) sp *= 2;
        const int64_t fine = std::min<int64_t>(1024 / units, p.Sk / 4096);
        if (fine > sp) sp = static_cast<int>(std::min<int64_t>(fine, 8));
    }
    p.splits = std::min(sp, std::max(1, blocks));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(attn_threads(D), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + pdl_attr(&attr[1], true);
    p.rtiles = 1;
    return launch_ranges(kern, cfg, p, "kv4 attention launch");
}

template <typename T>
int pick_attn(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    // Up to 8 rows fill this kernel's N side. 16 rows, here with two such tiles and
    // there: 16 sessions of 8192 slots of 4 heads, 64 channels 32.5 and 28.8 µs, 128
    // channels 49.5 and 34.3; one session of 2000 slots 6.5 and 6.5, 9.1 and 7.3 µs.
    if (p.R > kRows) return kv4tc::pick<T>(p, num_splits, s);
    return p.c.D == 64 ? launch_attn<T, 64>(p, num_splits, s) : launch_attn<T, 128>(p, num_splits, s);
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
    p.g = a.heads / p.c.Hkv; p.Sq = a.seq_q; p.Sk = a.seq_k; p.R = static_cast<int32_t>(R);
    p.causal = a.is_causal ? 1 : 0;
    p.sl2 = (a.scale == 0.f ? 1.f / sqrtf(static_cast<float>(p.c.D)) : a.scale) * 1.4426950408889634f;
    p.kv_len = a.kv_len; p.key_mask = a.key_mask; p.mask_sb = a.key_mask_stride_b;
    if (a.dtype == SFB_BF16) return kv4::pick_attn<__nv_bfloat16>(p, a.num_splits, s);
    return kv4::pick_attn<__half>(p, a.num_splits, s);
}

}  // namespace sfb
