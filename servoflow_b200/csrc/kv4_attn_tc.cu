// kv4_attn_tc.cu — attention over the 4-bit K/V cache on the 5th-generation
// tensor cores, for more than 8 rows per K/V head: an action chunk's
// cross-attention, a prompt chunk, grouped heads. kv4_attn.cu holds the
// form for few rows and the definitions (rows, masks, cache).
//
// As there, the keys are the MMA's M side. A tile is 128 keys by NQ rows:
//   Sᵀ[128 keys, NQ] = K · Qᵀ      A = K (fp16) in TMEM, B = Q in shared memory
//   Oᵀ[D, NQ]       += Vᵀ · Pᵀ     A = Vᵀ, B = Pᵀ, both in shared memory as the
//                                  rows of V and P lie (MN-major)
// 67 rows of an action chunk then cost 80 columns of exponentials (the bound: 16
// a clock per SM, 640 clocks a tile) instead of the 128 or 96 lanes that the
// rows cost as M. A thread of the softmax owns one key, so masks by length or
// key are one predicate per thread; a thread of the dequantisation owns one
// key's codes of 64 channels, 32 bytes of K and of V loaded a tile ahead, and
// writes K to its TMEM lane and V to its row of shared memory. K in TMEM rather than shared
// memory: the shared-memory port, at 128 B/clk, is the second bound (dequantised
// V 16 KB in and out, P 20 KB in and out, Q 10 KB out: 600 clocks a tile).
//
// Warps: a softmax group of four for every 16 columns (a thread then holds its
// key's logits and row sums in registers, S is read once and no column has two
// owners), four that dequantise for every 64 channels, one that issues the MMAs. Sᵀ and Pᵀ are double-
// buffered; Sᵀ of tile j + 2 is issued behind P·V of tile j, so that one barrier
// tells a group both that its logits are there and that its P buffer is free.
// The reference of a row (the m of exp2(x − m), kv4_attn.cu) is shared by a group's
// 128 threads through shared memory and raised only when a logit passes it by more
// than 15: a comparison a value with one vote of the group finds that out.
// (The vote of a tile cast one tile ahead, so that no warp waits for the others',
// takes the logits out of TMEM twice, or twice the registers: 32 sessions of 67
// rows by 4374 slots of 32 heads took 324 and 365 µs.)
//
// Measured: 32 sessions of 67 rows by 4374 slots, 32 heads of 64, 244 to 272 µs
// from one GPU to another (315 to 281 TFLOP/s); one session 15.4 µs; 8 sessions of 16
// heads of 128, 48 µs (399). A tile of 80 columns takes about 1900 clocks where the
// exponents alone are 640, one of 16 about 1450. What bounds it, by leaving parts out (64
// channels; µs, whole | without the softmax | without the loads of codes | without the
// softmax and all of the dequantisation but its barriers):
//   16 rows, 64 heads, 8192 slots       28.5 |  28.4 |  21.0 |  18.4
//   40 rows, 512 heads, 4374 slots     123   | 120   | 102   |  84
//   67 rows, 1024 heads, 4374 slots    266   | 244   | 237   | 164
//   96 rows, 128 heads, 4374 slots      40.3 |  34.9 |  38.1 |  24.7
// Few columns wait for the codes: the dequantising warps have one tile of them in
// flight. More columns wait for the softmax as well, neither chain hiding the other;
// the last column is the hand-overs between the warps, the MMAs, launch and join. One
// CTA per SM is all that TMEM, shared memory and registers allow.
//
// With M = 64 the accumulator's row d is in lane 32·(d / 16) + d % 16, with 128 in
// lane d.
// Every wait is bounded; an expired one records SFB_ERR_DEVICE_TIMEOUT.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sfb {
namespace kv4tc {

constexpr int kC = 16;                            // columns of a softmax group
__host__ __device__ constexpr int soft_warps(int nq) { return nq / kC * 4; }
__host__ __device__ constexpr int deq_warps(int d) { return d / 16; }   // four for every 64 channels
__host__ __device__ constexpr int threads(int d, int nq) { return (soft_warps(nq) + deq_warps(d) + 1) * 32; }   // + 1 issuing
constexpr int kMaxStages = 4;
__host__ __device__ constexpr int stages(int d) { return d == 64 ? 4 : 3; }   // dequantised K / V tiles
constexpr int kKeys = 128;
constexpr int kBlock64 = kKeys * 128;             // 64 channels of V, or 64 columns of P, of a tile
__host__ __device__ constexpr int max_q(int d) { return d == 64 ? 96 : 80; }
// TMEM columns: Sᵀ of tile j at 96·(j & 1), Oᵀ at 192, K (d / 2 columns a stage) at the end
constexpr int kTmemS = 0, kTmemO = 192;
__host__ __device__ constexpr int tmem_k(int d) { return 512 - stages(d) * (d / 2); }
__host__ __device__ constexpr int v_bytes(int d) { return d / 64 * kBlock64; }
constexpr int kOffQ = 0;                                      // [D / 64][max_q rows] × 128 B
__host__ __device__ constexpr int off_v(int d) { return d / 64 * max_q(d) * 128; }
__host__ __device__ constexpr int off_p(int d) { return off_v(d) + stages(d) * v_bytes(d); }     // [tile & 1][2 blocks]
__host__ __device__ constexpr int off_col(int d) { return off_p(d) + 2 * 2 * kBlock64; }       // per column: −m, m, alpha, limit
__host__ __device__ constexpr int off_bar(int d) { return off_col(d) + max_q(d) * 4 * (4 + 4); }   // and [4 windows] maxima, then row sums
constexpr int kNumBars = 2 * kMaxStages + 2 + 2 + 1 + 1 + 1;
__host__ __device__ constexpr int off_tmem(int d) { return off_bar(d) + 8 * kNumBars; }
__host__ __device__ constexpr int smem_bytes(int d) { return off_tmem(d) + 16 + 1024; }        // + alignment slack
__host__ __device__ constexpr bool layout_ok(int d) {
    // (more than half of an SM's: two kernels that take tensor memory never share one)
    return smem_bytes(d) <= 227 * 1024 && smem_bytes(d) > 114 * 1024 && kTmemO + max_q(d) <= tmem_k(d) && max_q(d) <= 128 && off_v(d) % 1024 == 0 &&
           off_p(d) % 1024 == 0 && off_col(d) % 16 == 0 && off_bar(d) % 8 == 0 &&
           // the partial result of a CTA, over P once every MMA is done: [NQ][D] O, [NQ] m, l
           max_q(d) * d * 4 + 2 * max_q(d) * 4 <= 4 * kBlock64;
}
static_assert(layout_ok(64) && layout_ok(128), "layout");

__host__ __device__ constexpr int bar_ready(int s) { return s; }                // K, V of a stage written
__host__ __device__ constexpr int bar_free(int s) { return kMaxStages + s; }       // both MMAs of a stage done
__host__ __device__ constexpr int bar_s(int u) { return 2 * kMaxStages + u; }      // Sᵀ of a tile, u = tile & 1
__host__ __device__ constexpr int bar_p(int u) { return 2 * kMaxStages + 2 + u; }  // Sᵀ read and Pᵀ written
constexpr int kBarO = 2 * kMaxStages + 4;                                          // P·V of a tile done
constexpr int kBarDone = kBarO + 1;                                                // P·V of the last tile done
constexpr int kBarDrain = kBarDone + 1;                                            // every MMA issued is done
constexpr float kUnseen = 1e30f;
constexpr uint64_t kWaitNs = 1000000000ull, kDrainNs = 100000000ull;

// 16 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
          "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr));
}
// Reduces 16 values per lane over the warp; the result of value i is left in the
// lanes with lane % 16 == i.
template <typename Op>
__device__ __forceinline__ float reduce16(float (&v)[16], int lane, Op op) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], 16));
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) {
        const bool up = (lane & w) != 0;
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const float send = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, w));
        }
    }
    return v[0];
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
// Barrier `id` of 128 threads with the OR of a predicate.
__device__ __forceinline__ bool bar_or(uint32_t id, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "barrier.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r) : "r"(x ? 1u : 0u), "r"(id) : "memory");
    return r != 0;
}
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(threads(D, NQ), 1) kv4_attn_tc_kernel(const Kv4AttnParams p) {
    using namespace ptx;
    constexpr int kSoftWarps = soft_warps(NQ), kSoftThreads = kSoftWarps * 32, kThreads = threads(D, NQ);
    constexpr int kDeqWarp0 = kSoftWarps, kCtrlWarp = kSoftWarps + deq_warps(D);
    constexpr int kMaxQ = max_q(D), kVBytes = v_bytes(D), kTmemK = tmem_k(D), kStages = stages(D);
    constexpr int kOffV = off_v(D), kOffP = off_p(D), kOffCol = off_col(D), kOffBar = off_bar(D), kOffTmem = off_tmem(D);
    static_assert(NQ <= kMaxQ && kThreads <= 1024, "columns");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // (stays a shared-memory address)
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + kOffTmem);
    float* negm = reinterpret_cast<float*>(smem + kOffCol);        // −m, kUnseen where no key was seen yet
    float* colm = negm + kMaxQ;
    float* alpha = colm + kMaxQ;
    int* lim = reinterpret_cast<int*>(alpha + kMaxQ);              // slots below lim[c] are visible to row c
    float* wred = alpha + 2 * kMaxQ;                               // [4 windows][kMaxQ]

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int split = blockIdx.x, hk = blockIdx.y / p.ytiles, rt = p.rt0 + blockIdx.y - hk * p.ytiles, b = blockIdx.z;
    // rows in equal tiles of at most NQ
    const int r0 = static_cast<int>(static_cast<int64_t>(p.R) * rt / p.rtiles);
    const int rows = static_cast<int>(static_cast<int64_t>(p.R) * (rt + 1) / p.rtiles) - r0;

    if (tid == kCtrlWarp * 32) {
        for (int s = 0; s < kStages; ++s) { mbar_init(&bars[bar_ready(s)], deq_warps(D)); mbar_init(&bars[bar_free(s)], 1); }
        for (int u = 0; u < 2; ++u) {
            mbar_init(&bars[bar_s(u)], 1);
            mbar_init(&bars[bar_p(u)], kSoftWarps);
        }
        mbar_init(&bars[kBarO], 1);
        mbar_init(&bars[kBarDone], 1);
        mbar_init(&bars[kBarDrain], 1);
        fence_mbarrier_init();
    }
    if (warp == 0) { tmem_alloc(tmem_holder, 512); tmem_relinquish(); }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_holder;
    pdl_trigger();                                 // TMEM is held: the next kernel may start
    pdl_wait();

    int n = p.Sk;
    if (p.kv_len != nullptr) n = min(n, max(0, p.kv_len[b]));
    auto limit = [&](int r) { return p.causal ? min(n, max(0, n - p.Sq + r / p.g + 1)) : n; };
    const int kend = limit(r0 + rows - 1), kfull = limit(r0);
    const int tiles = (kend + kKeys - 1) / kKeys;
    const int per = tiles / p.splits, rem = tiles - per * p.splits;
    const int t_begin = split * per + min(split, rem), ntl = per + (split < rem ? 1 : 0);
    const uint8_t* mask = p.key_mask != nullptr ? p.key_mask + b * p.mask_sb : nullptr;

    // ── Q (fp16, 128-byte-swizzled rows; zeros past the last row), columns ──
    bool bad = false;
    for (int i = tid; i < NQ * (D / 8); i += kThreads) {
        const int r = i / (D / 8), c = i % (D / 8);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const int rr = r0 + r, qi = rr / p.g, h = hk * p.g + (rr - qi * p.g);
            u = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_st[0] + h * p.q_st[1] +
                                                qi * p.q_st[2] + c * 8);
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    const float lo = __uint_as_float(w[e] << 16), hi = __uint_as_float(w[e] & 0xffff0000u);
                    bad |= (fabsf(lo) > 65504.f && !isinf(lo)) | (fabsf(hi) > 65504.f && !isinf(hi));
                    w[e] = kv4::h2u(__floats2half2_rn(lo, hi));
                }
                w[e] = kv4::inf_to_nan(w[e]);
                if (p.sl2 < 0.f) w[e] ^= 0x80008000u;      // the kernel's scale is |scale|
            }
        }
        *reinterpret_cast<uint4*>(smem + kOffQ + (c >> 3) * kMaxQ * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = u;
    }
    if (tid < NQ) {
        lim[tid] = tid < rows ? limit(r0 + tid) : kend;
        negm[tid] = kUnseen; colm[tid] = -INFINITY;
    }
    fence_proxy_async_smem();
    __syncthreads();

    bool ok = true;
    auto wait = [&](int bar, uint32_t parity) {
        if (mbar_try_wait(smem_u32(&bars[bar]), parity)) return;
        if (!ok || !mbar_wait(&bars[bar], parity, kWaitNs)) ok = false;
    };
    float* pO = reinterpret_cast<float*>(smem + kOffP);            // [NQ][D]
    float* pM = pO + kMaxQ * D;
    float* pL = pM + kMaxQ;

    if (warp >= kDeqWarp0 && warp < kCtrlWarp) {
        // ── dequantisation: thread = key and 64 channels of it ──────────────
        const int key_in = ((warp - kDeqWarp0) & 3) * 32 + lane, part = (warp - kDeqWarp0) >> 2;
        const uint32_t lane_off = static_cast<uint32_t>(((warp - kDeqWarp0) & 3) * 32) << 16;
        const int64_t first = static_cast<int64_t>(t_begin) * kKeys + key_in;
        int64_t co = b * p.c.code_sb + hk * p.c.code_sh + first * (D / 2) + part * 32;      // of the tile to load
        int64_t so = b * p.c.sc_sb + hk * p.c.sc_sh + (first * (D / 64) + part) * 2;
        int lkey = t_begin * kKeys + key_in;
        struct RawRow { uint4 k0, k1, v0, v1; __half2 ks, vs; };
        // a slot that is not seen is not read; its codes stand for 0 · 0
        auto load = [&](RawRow& r) {
            r.k0 = r.k1 = r.v0 = r.v1 = make_uint4(0, 0, 0, 0);
            r.ks = r.vs = __float2half2_rn(0.f);
            if (lkey < kend && (mask == nullptr || mask[lkey] != 0)) {
                const uint4* k4 = reinterpret_cast<const uint4*>(p.c.kc + co);
                const uint4* v4 = reinterpret_cast<const uint4*>(p.c.vc + co);
                r.k0 = k4[0]; r.k1 = k4[1]; r.v0 = v4[0]; r.v1 = v4[1];
                r.ks = *reinterpret_cast<const __half2*>(p.c.ks + so); r.vs = *reinterpret_cast<const __half2*>(p.c.vs + so);
            }
            co += kKeys * (D / 2); so += kKeys * (D / kv4::kGroup); lkey += kKeys;
        };
        RawRow nxt;
        if (ntl > 0) load(nxt);
        for (int j = 0; j < ntl; ++j) {
                RawRow r = nxt;
                if (j + 1 < ntl) load(nxt);
                if ((t_begin + j + 1) * kKeys > kfull) {           // slots that only some rows see
                    const int key = (t_begin + j) * kKeys + key_in;
                    if (key >= kfull && key < kend) {
                        kv4::contain(r.ks, r.vs);
                        if constexpr (D > 64) {                    // (the other half's V makes K NaN too)
                            __half2 v = *reinterpret_cast<const __half2*>(
                                p.c.vs + b * p.c.sc_sb + hk * p.c.sc_sh + (static_cast<int64_t>(key) * (D / 64) + 1 - part) * 2);
                            kv4::contain(r.ks, v);
                        }
                    }
                }
                const int s = j % kStages;
                if (j >= kStages) {
                    // (stages ahead of the MMAs: this wait is the long one, and not urgent)
                    if (!ok || !mbar_wait_sleep(&bars[bar_free(s)], ((j / kStages) - 1) & 1, 200, kWaitNs)) ok = false;
                    tc_fence_after_sync();
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 w = h ? r.k1 : r.k0;
                    const __half2 sc = h ? __high2half2(r.ks) : __low2half2(r.ks);
                    const uint32_t* wp = reinterpret_cast<const uint32_t*>(&w);
                    uint32_t kf[16];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t d4[4];
                        kv4::dequant_word(wp[x], sc, d4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) kf[4 * x + i] = d4[i];
                    }
                    tmem_st16(tmem + kTmemK + (D / 2) * s + 32 * part + 16 * h + lane_off, kf);
                }
                uint8_t* vrow = smem + kOffV + s * kVBytes + part * kBlock64 + key_in * 128;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 w = h ? r.v1 : r.v0;
                    const __half2 sc = h ? __high2half2(r.vs) : __low2half2(r.vs);
                    const uint32_t* wp = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t d4[4];
                        kv4::dequant_word(wp[x], sc, d4);
                        *reinterpret_cast<uint4*>(vrow + (((4 * h + x) ^ (key_in & 7)) << 4)) =
                            make_uint4(d4[0], d4[1], d4[2], d4[3]);
                    }
                }
                tmem_st_wait();
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[bar_ready(s)]);
        }
    } else if (warp == kCtrlWarp) {
        if (ntl > 0) {
            // ── MMA issue ───────────────────────────────────────────────────
            constexpr uint32_t idS = idesc_f16(128, NQ, 0, 0, 0);       // K(tmem) · Qᵀ, both K-major
            constexpr uint32_t idO = idesc_f16(D, NQ, 0, 1, 1);        // Vᵀ · Pᵀ, both MN-major
            const uint32_t aq = smem_u32(smem + kOffQ);
            auto issue_s = [&](int j) {
                const int s = j % kStages;
                tc_fence_after_sync();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        mma_f16_ts(tmem + kTmemS + 96 * (j & 1), tmem + kTmemK + (D / 2) * s + 8 * kk,
                                   smem_desc_sw128(aq + (kk >> 2) * kMaxQ * 128 + (kk & 3) * 32, 16, 1024), idS, kk > 0 ? 1u : 0u);
                    mma_commit(&bars[bar_s(j & 1)]);
                }
                __syncwarp();
            };
            auto issue_o = [&](int j) {
                const int s = j % kStages;
                tc_fence_after_sync();
                const uint32_t av = smem_u32(smem + kOffV + s * kVBytes);
                const uint32_t ap = smem_u32(smem + kOffP + (j & 1) * 2 * kBlock64);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_f16_ss(tmem + kTmemO, smem_desc_sw128(av + k * 2048, kBlock64, 1024),
                                   smem_desc_sw128(ap + k * 2048, kBlock64, 1024), idO, (j > 0 || k > 0) ? 1u : 0u);
                    mma_commit(&bars[bar_free(s)]);
                    mma_commit(&bars[kBarO]);
                }
                __syncwarp();
            };
            // (decisions are the whole warp's: a lane alone never leaves the loop)
            auto wait_all = [&](int bar, uint32_t parity) {
                if (!ok || !mbar_wait_sleep(&bars[bar], parity, 32, kWaitNs)) ok = false;   // none of these is urgent
                ok = __all_sync(0xffffffffu, ok) != 0;
                return ok;
            };
            for (int j = 0; j < min(2, ntl) && ok; ++j)
                if (wait_all(bar_ready(j), 0)) issue_s(j);
            // P·V of tile j before Sᵀ of tile j + 2, whose commit then also says that
            // tile j's buffer of P is free
            for (int j = 0; j < ntl && ok; ++j) {
                const int nx = j + 2;
                if (!wait_all(bar_p(j & 1), (j / 2) & 1)) break;
                issue_o(j);
                if (nx < ntl && wait_all(bar_ready(nx % kStages), (nx / kStages) & 1)) issue_s(nx);
            }
            // every MMA is done before TMEM and shared memory are let go
            if (elect_one()) {
                if (ok) mma_commit(&bars[kBarDone]);
                mma_commit(&bars[kBarDrain]);
            }
            __syncwarp();
            if (!mbar_wait(&bars[kBarDrain], 0, kDrainNs)) ok = false;
        }
    } else {
        // ── softmax: thread = key; group g has the columns [16·g, 16·g + 16) ──
        const int grp = warp >> 2, win = warp & 3, row = win * 32 + lane, c0 = kC * grp;
        const uint32_t lane_off = static_cast<uint32_t>(win * 32) << 16;
        const uint32_t tS = tmem + kTmemS + c0 + lane_off, tO = tmem + kTmemO + c0 + lane_off;
        const float sl2 = fabsf(p.sl2);
        const float2 s2 = make_float2(sl2, sl2);
        uint32_t poff[2];                          // this key's two 16-byte chunks (8 columns) in P's buffer
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = 2 * grp + i;
            poff[i] = kOffP + (c >> 3) * kBlock64 + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        }
        float2 l[kC / 2];
#pragma unroll
        for (int i = 0; i < kC / 2; ++i) l[i] = make_float2(0.f, 0.f);
        for (int j = 0; j < ntl; ++j) {
            const int k0 = (t_begin + j) * kKeys, key = k0 + row, u = j & 1;
            const bool edge = k0 + kKeys > kfull || mask != nullptr;
            wait(bar_s(u), (j / 2) & 1);           // also: P·V of tile j − 2 is done, its P buffer free
            tc_fence_after_sync();
            float x[kC];
            tmem_ld16(tS + 96 * u, x);
            tmem_ld_wait();
            auto hide = [&]() {                    // keys that some row does not see
                const bool vis = key < kend && (mask == nullptr || mask[key] != 0);
#pragma unroll
                for (int i = 0; i < kC; ++i) x[i] = vis && key < lim[c0 + i] ? x[i] : -INFINITY;
            };
            auto to_exponents = [&]() {            // x → x·sl2 − m
#pragma unroll
                for (int i = 0; i < kC; i += 4) {
                    const float4 m4 = *reinterpret_cast<const float4*>(negm + c0 + i);
                    const float2 t0 = fma2(make_float2(x[i], x[i + 1]), s2, make_float2(m4.x, m4.y));
                    const float2 t1 = fma2(make_float2(x[i + 2], x[i + 3]), s2, make_float2(m4.z, m4.w));
                    x[i] = t0.x; x[i + 1] = t0.y; x[i + 2] = t1.x; x[i + 3] = t1.y;
                }
            };
            if (edge) hide();
            to_exponents();
            // does any logit pass its row's reference by more than kOver? (a row that saw
            // no key yet has the reference −kUnseen)
            float over[2] = {x[0], x[1]};
#pragma unroll
            for (int i = 2; i < kC; i += 2) over[(i / 2) & 1] = fmaxf(fmaxf(over[(i / 2) & 1], x[i]), x[i + 1]);
            if (bar_or(1 + grp, fmaxf(over[0], over[1]) > kv4::kOver)) {
                // raise the references: column maxima of the tile, over a warp's keys, then its group's warps
                tmem_ld16(tS + 96 * u, x);
                tmem_ld_wait();
                if (edge) hide();
                {
                    const float mx = reduce16(x, lane, [](float a, float c) { return fmaxf(a, c); });
                    if (lane < kC) wred[win * kMaxQ + c0 + lane] = mx;
                }
                named_bar_sync(1 + grp, 128);
                if (row < kC) {
                    const float* cm = wred + c0 + row;
                    const float t = fmaxf(fmaxf(cm[0], cm[kMaxQ]), fmaxf(cm[2 * kMaxQ], cm[3 * kMaxQ])) * sl2;
                    const float old = colm[c0 + row];
                    float al = 1.f;
                    if (t > old + kv4::kOver) {
                        const float m = t - kv4::kBelow;
                        al = old == -INFINITY ? 0.f : ex2(old - m);
                        colm[c0 + row] = m;
                        negm[c0 + row] = -m;
                    }
                    alpha[c0 + row] = al;
                }
                named_bar_sync(1 + grp, 128);
#pragma unroll
                for (int i = 0; i < kC / 2; ++i) {
                    const float2 al = *reinterpret_cast<const float2*>(alpha + c0 + 2 * i);
                    l[i].x *= al.x; l[i].y *= al.y;
                }
                if (j > 0) {
                    // the accumulator is at rest (P·V of tile j − 2 is done, its commit
                    // came before that of S: one phase at most is open)
                    wait(kBarO, (j - 1) & 1);
                    tc_fence_after_sync();
                    float a[kC];
                    tmem_ld16(tO, a);
                    tmem_ld_wait();
                    uint32_t w[kC];
#pragma unroll
                    for (int i = 0; i < kC; ++i) w[i] = __float_as_uint(a[i] * alpha[c0 + i]);
                    tmem_st16(tO, w);
                    tmem_st_wait();
                }
                named_bar_sync(1 + grp, 128);                       // alpha is read before it is written again
                tmem_ld16(tS + 96 * u, x);                          // (again: registers)
                tmem_ld_wait();
                if (edge) hide();
                to_exponents();
            }
            // P = 2^(x·sl2 − m), row sums, fp16 P into this key's row
#pragma unroll
            for (int i = 0; i < kC; i += 8) {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 p0 = make_float2(ex2(x[i + e]), ex2(x[i + e + 1]));
                    l[(i + e) / 2] = add2(l[(i + e) / 2], p0);
                    h[e / 2] = kv4::h2u(__floats2half2_rn(p0.x, p0.y));
                }
                *reinterpret_cast<uint4*>(smem + poff[i / 8] + u * 2 * kBlock64) = make_uint4(h[0], h[1], h[2], h[3]);
            }
            fence_proxy_async_smem();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[bar_p(u)]);
        }
        // row sums over the warp's keys
        {
            float v[kC];
#pragma unroll
            for (int i = 0; i < kC; ++i) v[i] = (i & 1) ? l[i / 2].y : l[i / 2].x;
            const float t = reduce16(v, lane, [](float a, float c) { return a + c; });
            if (lane < kC) wred[win * kMaxQ + c0 + lane] = t;
        }
        // every P·V is done: P's memory becomes the partial result. kBarDone has one
        // phase. kBarO cannot say this: here P·V of tile ntl − 3 is known to be done
        // (S of tile ntl − 1 was committed behind it) and no later one, so kBarO may be
        // two phases short of ntl, where a wait for the last one's parity is answered
        // by the phase two before it.
        if (ntl > 0) wait(kBarDone, 0);
        tc_fence_after_sync();
        named_bar_sync(7, kSoftThreads);
        {
            // with M = 64 lanes 0..15 hold row d of Oᵀ, with 128 all do
            const int d = D == 64 ? 16 * win + (lane & 15) : row;
            float a[kC];
            tmem_ld16(tO, a);
            tmem_ld_wait();
            if (D > 64 || lane < 16) {
#pragma unroll
                for (int i = 0; i < kC; ++i) pO[(c0 + i) * D + d] = ntl > 0 ? a[i] : 0.f;
            }
            if (row < kC) {
                const float* ls = wred + c0 + row;
                pM[c0 + row] = colm[c0 + row];
                pL[c0 + row] = (ls[0] + ls[kMaxQ]) + (ls[2 * kMaxQ] + ls[3 * kMaxQ]);
            }
        }
        named_bar_sync(7, kSoftThreads);
        T* out = static_cast<T*>(p.out);
        auto store = [&](int r, int d, float4 a, float inv) {
            const int rr = r0 + r, qi = rr / p.g, h = hk * p.g + (rr - qi * p.g);
            T* dst = out + b * p.o_st[0] + h * p.o_st[1] + qi * p.o_st[2] + d;
            uint2 u;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
                u.x = *reinterpret_cast<const uint32_t*>(&x); u.y = *reinterpret_cast<const uint32_t*>(&y);
            } else {
                u.x = kv4::h2u(__floats2half2_rn(a.x * inv, a.y * inv)); u.y = kv4::h2u(__floats2half2_rn(a.z * inv, a.w * inv));
            }
            *reinterpret_cast<uint2*>(dst) = u;
        };
        if (p.splits == 1) {
            // (with every logit of a row NaN its sum is, and so is the row)
            if (ok)
                for (int i = tid; i < rows * (D / 4); i += kSoftThreads) {
                    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
                    const float L = pL[r];
                    store(r, d, *reinterpret_cast<const float4*>(pO + r * D + d), L != 0.f ? 1.f / L : 0.f);
                }
        } else {
            cluster_sync();                        // every CTA's partial is written
            const uint32_t aO = smem_u32(pO), aM = smem_u32(pM), aL = smem_u32(pL);
            const int mine = split < rows ? (rows - split + p.splits - 1) / p.splits : 0;
            for (int i = tid; i < mine * (D / 4); i += kSoftThreads) {
                const int r = split + (i / (D / 4)) * p.splits, d = (i % (D / 4)) * 4;
                float M = -INFINITY, L = 0.f;
                for (int k = 0; k < p.splits; ++k) M = fmaxf(M, dsmem_ld_f32(dsmem_map(aM + 4 * r, k)));
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < p.splits; ++k) {
                    const float mk = dsmem_ld_f32(dsmem_map(aM + 4 * r, k)), lk = dsmem_ld_f32(dsmem_map(aL + 4 * r, k));
                    if (mk == -INFINITY) { L += lk; continue; }
                    const float f = ex2(mk - M);
                    L += f * lk;
                    const float4 v = dsmem_ld_f32x4(dsmem_map(aO + 4 * (r * D + d), k));
                    a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
                }
                if (ok) store(r, d, a, L != 0.f ? 1.f / L : 0.f);
            }
            cluster_sync();                        // nobody leaves while its partial may be read
        }
    }
    if (warp >= kSoftWarps && p.splits > 1) { cluster_sync(); cluster_sync(); }
    if (bad) atomicExch(&g_sfb_device_error, SFB_ERR_RANGE);
    if (!ok) atomicExch(&g_sfb_device_error, SFB_ERR_DEVICE_TIMEOUT);
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int D, int NQ>
int launch(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    const DeviceInfo& dev = device_info();
    auto kern = kv4_attn_tc_kernel<T, D, NQ>;
    static std::atomic<bool> done[64];             // kernel attributes, once per device (idempotent)
    if (!done[dev.ordinal & 63].load(std::memory_order_acquire)) {
        const cudaError_t e1 = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(D));
        const cudaError_t e2 = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e1 != cudaSuccess || e2 != cudaSuccess) {
            record_cuda_error(e1 != cudaSuccess ? e1 : e2, "kv4 attention attributes");
            return SFB_ERR_CUDA;
        }
        prefer_max_shared(kern);
        done[dev.ordinal & 63].store(true, std::memory_order_release);
    }
    p.rtiles = (p.R + NQ - 1) / NQ;
    const int64_t units = static_cast<int64_t>(p.c.B) * p.c.Hkv * p.rtiles;
    const int tiles = (p.Sk + kKeys - 1) / kKeys;
    int sp = num_splits;
    if (sp == 0) {
        // as many as keep every CTA in one wave (one per SM), two tiles each at least.
        // (More, where one wave is passed by little: 176 row tiles of 17 key tiles took
        // 54 µs in three rounds of halves, 48 in two rounds.)
        sp = static_cast<int>(std::min<int64_t>(16, std::max<int64_t>(1, dev.num_sms / units)));
        sp = std::min(sp, std::max(1, tiles / 2));
    }
    p.splits = std::min(sp, std::max(1, tiles));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(threads(D, NQ), 1, 1);
    cfg.dynamicSmemBytes = smem_bytes(D);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1 + pdl_attr(&attr[1], true);
    return kv4::launch_ranges(kern, cfg, p, "kv4 attention (tcgen05) launch");
}

// The column count that takes the least time: rounds of the SMs (or the share of a
// round that splitting a CTA's keys leaves) times a tile's, which grows as nq + 88
// (16 × 32 units of 40 rows: 126 µs with 48 columns, 150 with 80; 2060 rows of 8
// units: 43.6 µs with 80, 47.7 with 96, 51.9 with 48; 67 rows of 32 units: 15.6 µs
// with 80, 17.7 with 48, of 1024 units 271 and 427).
template <typename T>
int pick(Kv4AttnParams& p, int num_splits, cudaStream_t s) {
    if (p.R <= 16) return p.c.D == 128 ? launch<T, 128, 16>(p, num_splits, s) : launch<T, 64, 16>(p, num_splits, s);
    const int64_t sms = std::max(device_info().num_sms, 1);
    auto cost = [&](int nq) {
        const int64_t units = std::max<int64_t>(1, static_cast<int64_t>((p.R + nq - 1) / nq) * p.c.B * p.c.Hkv);
        const double rounds = units <= sms ? 1.0 / std::min<int64_t>(16, sms / units) : static_cast<double>((units + sms - 1) / sms);
        return rounds * (nq + 88);
    };
    const double c48 = cost(48), c80 = cost(80), c96 = cost(96);
    if (p.c.D == 128) return c80 <= c48 ? launch<T, 128, 80>(p, num_splits, s) : launch<T, 128, 48>(p, num_splits, s);
    if (c96 <= c80 && c96 <= c48) return launch<T, 64, 96>(p, num_splits, s);
    if (c80 <= c48) return launch<T, 64, 80>(p, num_splits, s);
    return launch<T, 64, 48>(p, num_splits, s);
}

}  // namespace kv4tc
}  // namespace sfb
