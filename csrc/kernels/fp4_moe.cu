// A whole layer of 4-bit experts for a few tokens (1..32) in two kernels.
//
//   p = score(logits), chosen = top-k of p + bias (in f32; ties to the lower index), w = scale * p / sum(chosen p)
//   g, u = W13[e] . e4m3(x)                            e4m3(.): power-of-two scale per 32 values
//   h[e, t] = e4m3(silu(min(g, limit)) * clamp(u, -limit, limit) * w[t, e])
//   y[t] = sum over chosen e of W2[e] . h[e, t]
//
// The layer is bound by streaming the chosen experts' weights (17/32 byte per value) once.  Nothing is dequantised in
// registers: tcgen05.mma kind::mxf8f6f4.block_scale multiplies e2m1 weights with e4m3 activations and applies both
// scale vectors; the padded 4-bit form that it wants in shared memory (16 codes in 8 bytes, 8 bytes of gap) is what a TMA
// box of the 4-bit element type writes, so weight bytes go from HBM to the tensor core without passing a register.
// The weights are the operand on the 128 lanes, ALL tokens (padded to 8, 16 or 32) are the columns, for every expert that any
// token chose: columns of tokens that did not choose the expert cost no bytes, and are dropped (gate | up) or zero (down).
//
// Kernel 1 (gate_up): persistent clusters of S CTAs.  Every CTA routes all tokens by itself (a warp per token; the logits
// are a few KB in L2, and a separate routing launch costs more), quantises its K range of x into shared memory once, and
// walks the (expert, 128 rows of I) tiles of its cluster, each CTA over 1/S of K.  The S partial sums of a 32-row
// quarter meet in the CTA that owns the quarter (pushed through distributed shared memory, summed in rank order), which
// applies SwiGLU and quantises: 32 rows of a lane quarter are exactly one block of h.  h is stored in the swizzled
// operand form, so kernel 2 fetches it with plain bulk copies.
// Kernel 2 (down): a cluster of S CTAs per 128 rows of the output; the (expert, 128 columns of I) blocks of all chosen
// experts are one long K axis, split over the cluster, accumulated in ONE accumulator: the sum over experts costs
// nothing.  Partials are summed in rank order.  No atomics anywhere: the same bits every run.
// Both kernels are launched with programmatic serialisation: they set up (barriers, tables) beside the end of the kernel
// before and wait for it before they read anything (one token, call after call: 36.9 us without it for kernel 1, 34.6 with).
// Kernel 2 then reads the list of chosen experts, which kernel 1 leaves behind (routing again there cost 4 us at its head).
// Experts of 5120 x 2304, a call among others: one token (6 experts, 113 MB, 17.2 us of HBM) 34 us: 7 until the first weight of kernel 1
// (routing 5), 12.5 of weights, 5 until the first weight of kernel 2, 5 of weights, 2 for the sum; 5 tokens (15 experts, 43 us of HBM)
// 59 us; 32 tokens (88 experts, 252 us of HBM) 320 us, 18 of them routing.  8 tokens of 44 experts of 5120 x 576 (32 us of HBM)
// 60 us.  The first kernel's weights in flight decide at 32 tokens: six stages beside x and the receive slots 338 us, seven 317.
#include "fp4_common.cuh"

namespace {

using namespace fp4;

constexpr int kMaxE = 512, kMaxTok = 32, kMaxTopk = 32;
constexpr int kUpThreads = 640, kRouteThreads = 256;   // kernel 1: warps 0..7 route, the others quantise x meanwhile
constexpr int kDownThreads = 320;

enum Score : int { kSqrtSoftplus = 0, kSigmoid = 1, kSoftmax = 2 };

struct MoeArgs {
    const void* x;
    int64_t ldx;
    const float *logits, *bias;
    int64_t ldl;
    const uint8_t *s13, *s2;
    void* out;
    int64_t ldo;
    uint8_t *h, *hs;          // [active][nit][BN * 128] operand tiles, [active][nit][512] their scale chunks
    int* list;                // number of chosen experts, then the experts, ascending
    float scale, limit;
    int xdt, odt, accumulate, T, E, topk, D, I, score, norm;
    int g1, nit, S;           // 128-column groups of D, 128-row tiles of I, cluster size
    int* status;
};

struct Route {
    uint32_t mask[kMaxE];                     // tokens that chose the expert
    float wt[kMaxTok * kMaxTopk];
    uint16_t sel[kMaxTok * kMaxTopk];
    uint16_t act[kMaxE];                      // chosen experts, ascending
    float mx[kMaxTok], inv[kMaxTok];          // softmax: largest logit, 1 / sum
    int n_act, next;
};

__device__ __forceinline__ uint32_t order_key(float v) {   // larger float -> larger key; NaN below every number; 0 is free
    if (v != v) return 1u;
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float score_of(float z, int score, float mx, float inv_sum) {
    if (score == kSigmoid) return 1.f / (1.f + expf(-z));
    if (score == kSoftmax) return expf(z - mx) * inv_sum;
    return sqrtf(fmaxf(z, 0.f) + log1pf(expf(-fabsf(z))));
}

// Routing.  Every CTA does it once, before its first weight arrives: what counts is the length of the dependent chain and
// the size of the code (straight-line code that runs once costs its instruction fetches: with the scores unrolled over a
// lane's 16 experts it took 30 us for one token), so the score loops are rolled and the selection is a tree over registers.
// From eight tokens on a warp takes a token at a time; below, the first kRouteThreads threads share the scores.

// Logits of token t to row (shared memory); for softmax its largest logit and 1 / sum.  One warp.
__device__ __forceinline__ void route_load(const MoeArgs& a, Route& r, float* row, int t, int lane) {
    constexpr int kPer = kMaxE / 32;
    float z[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) z[j] = lane + 32 * j < a.E ? ld_f32(a.logits + t * a.ldl + lane + 32 * j) : -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (lane + 32 * j < a.E) row[lane + 32 * j] = z[j];
    if (a.score == kSoftmax) {
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) mx = fmaxf(mx, z[j]);
        mx = warp_max(mx);
        if (mx == -INFINITY) mx = 0.f;
        __syncwarp();
#pragma unroll 1
        for (int e = lane; e < a.E; e += 32) sum += expf(row[e] - mx);
        sum = warp_sum(sum);
        if (lane == 0) { r.mx[t] = mx; r.inv[t] = 1.f / sum; }
    }
}
// Keys of the row's logits, from expert `first` in steps of `step` (with a bias; without, the logit itself decides, exactly:
// every score grows with its logit).  They may take the logits' place.
__device__ __forceinline__ void route_keys(const MoeArgs& a, const Route& r, const float* row, float* keys, const float* bias, int t,
                                           int first, int step) {
    const float mx = r.mx[t], inv = r.inv[t];
#pragma unroll 1
    for (int e = first; e < a.E; e += step)
        reinterpret_cast<uint32_t*>(keys)[e] = order_key(score_of(row[e], a.score, mx, inv) + bias[e]);
}
// The token's choice from its row of keys (or, without a bias, of logits); z: its logits.  One warp.
__device__ __forceinline__ void route_pick(const MoeArgs& a, Route& r, const float* row, const volatile float* z, int t, int lane) {
    constexpr int kPer = kMaxE / 32;
    uint32_t key[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int e = lane + 32 * j;
        key[j] = e >= a.E ? 0u : a.bias ? __float_as_uint(row[e]) : order_key(row[e]);
    }
    int mine = 0;
    float p = 0.f;
#pragma unroll 1
    for (int k = 0; k < a.topk; ++k) {
        uint32_t m[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) m[j] = key[j];
#pragma unroll
        for (int o = kPer / 2; o > 0; o >>= 1)
#pragma unroll
            for (int j = 0; j < o; ++j) m[j] = max(m[j], m[j + o]);
        const uint32_t top = __reduce_max_sync(0xffffffffu, m[0]);
        uint32_t hit = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) hit |= key[j] == top ? 1u << j : 0u;
        const uint32_t cand = hit ? (uint32_t)(lane + 32 * (__ffs(hit) - 1)) : 0xffffffffu;
        const uint32_t e = __reduce_min_sync(0xffffffffu, cand);
        if (lane == k) {
            mine = (int)e;
            p = z[e];   // in flight over the rounds that follow
        }
        const uint32_t gone = (e & 31u) == (uint32_t)lane ? 1u << (e >> 5) : 0u;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (gone >> j & 1) key[j] = 0u;
    }
    p = lane < a.topk ? score_of(p, a.score, r.mx[t], r.inv[t]) : 0.f;
    if (a.norm) {   // scores are not negative: a sum of zero is all of them zero
        const float sum = warp_sum(p);
        p = sum == 0.f ? 0.f : p / sum;
    }
    if (lane < a.topk) {
        r.sel[t * kMaxTopk + lane] = (uint16_t)mine;
        r.wt[t * kMaxTopk + lane] = p * a.scale;
        atomicOr(&r.mask[mine], 1u << t);
    }
}
// Few tokens: the first kRouteThreads threads.  Scratch: the bias, a row of logits per token, a row of keys per token.
__device__ __forceinline__ void route_together(const MoeArgs& a, Route& r, float* bias) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int nw = kRouteThreads / 32;
    float *rows = bias + a.E, *keys = rows + a.T * a.E;
    auto sync = [&]() { asm volatile("bar.sync 2, %0;" ::"n"(kRouteThreads) : "memory"); };
    if (warp < a.T) {
        route_load(a, r, rows + warp * a.E, warp, lane);
    } else if (a.bias) {   // (a.T < nw: the loads of logits and bias fly together)
#pragma unroll 4
        for (int e = (warp - a.T) * 32 + lane; e < a.E; e += (nw - a.T) * 32) bias[e] = ld_f32(a.bias + e);
    }
    if (a.bias) {
        sync();
        const int stripes = nw / a.T;
        if (warp < a.T * stripes) {
            const int t = warp / stripes;
            route_keys(a, r, rows + t * a.E, keys + t * a.E, bias, t, (warp - t * stripes) * 32 + lane, 32 * stripes);
        }
        sync();
    }
    __syncwarp();
    if (warp < a.T) route_pick(a, r, (a.bias ? keys : rows) + warp * a.E, rows + warp * a.E, warp, lane);
}
// Many tokens: any warp, the next token that nobody has taken.
__device__ __forceinline__ void route_in_turn(const MoeArgs& a, Route& r, const float* bias, float* rows) {
    const int lane = threadIdx.x & 31;
    for (;;) {
        int t = 0;
        if (lane == 0) t = atomicAdd(&r.next, 1);
        t = __shfl_sync(0xffffffffu, t, 0);
        if (t >= a.T) break;
        float* row = rows + t * a.E;
        route_load(a, r, row, t, lane);
        __syncwarp();
        if (a.bias) route_keys(a, r, row, row, bias, t, lane, 32);
        __syncwarp();
        route_pick(a, r, row, a.logits + t * a.ldl, t, lane);
    }
}
// The chosen experts, ascending, to r.act and (block 0) to kernel 2.  One warp, after all choices.
__device__ __forceinline__ void route_list(const MoeArgs& a, Route& r, int lane) {
    constexpr int kPer = kMaxE / 32;
    uint32_t on[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) on[j] = __ballot_sync(0xffffffffu, r.mask[lane + 32 * j] != 0u);
    int n = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (on[j] >> lane & 1) r.act[n + __popc(on[j] & ((1u << lane) - 1u))] = (uint16_t)(lane + 32 * j);
        n += __popc(on[j]);
    }
    if (lane == 0) r.n_act = n;
    __syncwarp();
    if (blockIdx.x == 0) {
        for (int i = lane; i < n; i += 32) a.list[1 + i] = r.act[i];
        if (lane == 0) a.list[0] = n;
    }
}

// kind::mxf8f6f4: A e2m1 (5), B e4m3 (0), ue8m0 scales, M = 128
__host__ __device__ constexpr uint32_t moe_idesc(int N, int sf) {
    return ((uint32_t)sf << 4) | (5u << 7) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24) | ((uint32_t)sf << 29);
}
__device__ __forceinline__ void umma_w4a8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
}
// The four MMAs of a 128-column block.
template <int BN>
__device__ __forceinline__ void mma_block(uint32_t d, uint64_t w, uint64_t x, uint32_t sfw, uint32_t sfx, bool accumulate) {
#pragma unroll
    for (int k = 0; k < 4; ++k) umma_w4a8(d, w + 2u * k, x + 2u * k, moe_idesc(BN, k), sfw, sfx, accumulate || k ? 1u : 0u);
}
// Both stages full (the second only if `two`).  The tensor core holds few MMAs in its queue, so it idles while this thread waits
// (about 75 clocks, against 156 for a block's four MMAs): two blocks per wait.
__device__ __forceinline__ bool wait_two(uint32_t bar0, uint32_t par0, uint32_t bar1, uint32_t par1, bool two) {
    const bool r0 = tc::mbar_try_wait(bar0, par0), r1 = !two || tc::mbar_try_wait(bar1, par1);
    const bool ok = (r0 || tc::mbar_wait(bar0, par0)) && (r1 || tc::mbar_wait(bar1, par1));
    tc::tc_fence_after();
    return ok;
}
__device__ __forceinline__ void tmem_ld1(uint32_t taddr, float& v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(v) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, float (&v)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, long long budget = 2000000000ll) {
    const long long t0 = clock64();
    for (;;) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (clock64() - t0 > budget) return false;
    }
}

template <int BN>
struct UpCfg {
    static constexpr int kA = 128 * 128;                       // padded 4-bit tile: one matrix, 128 columns
    static constexpr int kStage = kA + 512;                    // and its scale chunk (kept apart: tiles start on 1024 bytes)
    static constexpr int kAccSet = 2 * BN;                     // gate | up columns of one accumulator set
    static constexpr int kSfW = 2 * kAccSet, kSfX = kSfW + 8;  // scales: 2 x 4 columns of weights, 4 per block of x (an
                                                               // MMA takes its scales from a multiple of four columns)
    static constexpr int kTmem = 512;
    static constexpr int kBars = 512;
    static constexpr int kMaxKb = 64;                          // 128-column blocks of x per CTA
    static_assert(kSfX + 4 * kMaxKb <= kTmem, "tensor memory");
};

// Shared memory of kernel 1: x blocks | their scale chunks, then receive slots | stages | stage scales | barriers.  The scale
// chunks are in tensor memory before the first tile is through, so the slots may take their place once the owner says so
// (32 tokens, 5120 columns, S = 2: seven stages instead of six).
template <int BN>
__host__ __device__ constexpr size_t up_recv_bytes(int S) { return S == 1 ? 0 : (size_t)(S - 1) * (S >= 4 ? 1 : 4 / S) * 2 * BN * 128; }
template <int BN>
__host__ __device__ constexpr size_t up_front(int nkb, int S) {
    const size_t sf = (size_t)nkb * 512, recv = up_recv_bytes<BN>(S);
    return ((size_t)nkb * BN * 128 + (sf > recv ? sf : recv) + 1023) / 1024 * 1024;
}
template <int BN>
__host__ __device__ constexpr size_t up_fixed(int nkb, int S) { return up_front<BN>(nkb, S) + 1024 + UpCfg<BN>::kBars; }

template <int BN, typename TX>
__global__ void __launch_bounds__(kUpThreads, 1)
fp4_moe_up_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_tail, const MoeArgs a, int stages) {
    using C = UpCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Route R;
    __shared__ int s_fail;
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_g = smem_raw + (base - tc::smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = a.S, rank = S > 1 ? (int)cluster_rank() : 0;
    const int kb0 = a.g1 * rank / S, kb1 = a.g1 * (rank + 1) / S, nkb = kb1 - kb0;
    const int nkb_max = (a.g1 + S - 1) / S;
    const uint32_t xsf_off = (uint32_t)nkb_max * BN * 128;
    const uint32_t recv_off = xsf_off;
    const uint32_t st_off = (uint32_t)up_front<BN>(nkb_max, S);
    const uint32_t sf_off = st_off + (uint32_t)stages * C::kA;
    const uint32_t bars = base + sf_off + (uint32_t)stages * 512;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (stages + s); };
    const uint32_t acc_full = bars + 16u * stages, acc_empty = acc_full + 16u, recv_full = acc_empty + 16u, recv_free = recv_full + 32u,
                   tmem_slot = recv_free + 32u;

    if (warp == 9) {
        if (lane == 0) {
            s_fail = 0;
            for (int s = 0; s < stages; ++s) {
                tc::mbar_init(full(s), 1);
                tc::mbar_init(empty(s), 1);
            }
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(acc_full + 8u * i, 1);
                tc::mbar_init(acc_empty + 8u * i, 4);
            }
            for (int q = 0; q < 4; ++q) {
                tc::mbar_init(recv_full + 8u * q, S > 1 ? S - 1 : 1);
                tc::mbar_init(recv_free + 8u * q, 1);
            }
            tc::mbar_fence_init();
            tc::prefetch_tmap(&tmap_w);
            tc::prefetch_tmap(&tmap_tail);
        }
    }
    float* scratch = reinterpret_cast<float*>(base_g + st_off);   // of the routing, where the first weights will land
    const bool few = a.T < kRouteThreads / 32;
    for (int e = threadIdx.x; e < kMaxE; e += kUpThreads) R.mask[e] = 0u;
    if (threadIdx.x == 0) R.next = 0;
    __syncthreads();
    pdl_wait();   // everything below reads what may come from the kernel before
    if (!few && a.bias) {
        for (int e = threadIdx.x; e < a.E; e += kUpThreads) scratch[e] = ld_f32(a.bias + e);
        __syncthreads();
    }
    if (threadIdx.x < kRouteThreads) {
        if (few) route_together(a, R, scratch);
    } else {
        // ---- this CTA's K range of x, quantised, in operand form ----
        const TX* x = reinterpret_cast<const TX*>(a.x);
        const bool vec = (uintptr_t)x % (8 * sizeof(TX)) == 0 && a.ldx % 8 == 0;
        constexpr int kN = kUpThreads - kRouteThreads, kBatch = 4;
        // e4m3 of eight values (m: the largest |.|) to their place in row t; a block of 32 columns is four lanes
        auto put = [&](int t, int c, bool in, const float (&v)[8], uint32_t m) {
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const uint32_t sb = ue8m0_of(m, 1e-4f, kInv448);
            const float inv = sb == 255u ? 0.f : ue8m0_inv(sb);
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
                w[i] = sb == 255u ? 0u : lo | hi << 16;
            }
            if (in) {
                const int kb = c >> 4, u16 = c & 15;       // u16: 8-byte unit of the 128-byte row
                *reinterpret_cast<uint2*>(base_g + kb * (BN * 128) + t * 128 + (((u16 >> 1) ^ (t & 7)) << 4) + (u16 & 1) * 8) = make_uint2(w[0], w[1]);
                if ((c & 3) == 0) base_g[xsf_off + kb * 512 + t * 16 + (u16 >> 2)] = (uint8_t)sb;
            }
        };
        const int tid = threadIdx.x - kRouteThreads, per_row = nkb * 16;      // units of eight columns
        if (vec && kb1 * 128 <= a.D) {
            // a thread keeps its eight columns over the tokens, the next four tokens' loads in flight
#pragma unroll 1
            for (int c0 = 0; c0 < per_row; c0 += kN) {
                const int c = c0 + tid;
                const bool in = c < per_row;
                const TX* xc = x + kb0 * 128 + (in ? c : 0) * 8;
                Raw8<TX> cur[kBatch], nxt[kBatch];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) cur[b].load(xc + min(b, a.T - 1) * a.ldx);
#pragma unroll 1
                for (int t0 = 0; t0 < a.T; t0 += kBatch) {
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) nxt[b].load(xc + min(t0 + kBatch + b, a.T - 1) * a.ldx);
#pragma unroll
                    for (int b = 0; b < kBatch; ++b)
                        if (t0 + b < a.T) {
                            float v[8];
                            cur[b].unpack(v);
                            put(t0 + b, c, in, v, cur[b].max_bits());
                        }
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) cur[b] = nxt[b];
                }
            }
        } else {
#pragma unroll 1
            for (int c0 = 0; c0 < per_row; c0 += kN) {
                const int c = c0 + tid, col = kb0 * 128 + c * 8;
                const bool in = c < per_row;
#pragma unroll 1
                for (int t = 0; t < a.T; ++t) {
                    float v[8];
                    load8(x + t * a.ldx + min(col, a.D - 1), in ? max(0, min(8, a.D - col)) : 0, false, v);
                    put(t, c, in, v, max_bits8(v));
                }
            }
        }
    }
    if (!few) route_in_turn(a, R, scratch, scratch + a.E);   // (warps that quantised x join when they are through)
    __syncwarp();
    if (warp == 9) {
        tc::tmem_alloc(tmem_slot, C::kTmem);
        pdl_launch();   // not before: a dependent on this SM could take the tensor memory first, and waits for this kernel's end
    }
    fence_proxy_async();                         // x blocks, and the scratch that becomes the target of TMA copies
    __syncthreads();
    if (warp == 0) route_list(a, R, lane);
    __syncwarp();
    tc::tc_fence_before();
    if (S > 1) cluster_sync_all(); else __syncthreads();
    tc::tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

    const int items = R.n_act * a.nit;
    const int first = blockIdx.x / S, step = gridDim.x / S;

    if (warp == 0 || warp == 6) {
        if (elect_one()) {
            // Two producers take turns: one thread needs about 310 clocks for a block's wait, count and two copies, more than
            // the block's MMAs.  Stage and how often the ring went round are counted, not divided for.
            const int mine = warp == 6;
            int s = mine, round = 0, it = 0;
            bool ok = true;
            for (int item = first; item < items && ok; item += step) {
                const int e = R.act[item / a.nit], j = item % a.nit;
                const int rows = min(128, a.I - j * 128), boxes = rows == 128 ? 0 : (rows + 31) / 32;
                int row = (e * 2) * a.I + j * 128;
                const uint8_t* sf = a.s13 + (((int64_t)e * 2) * a.nit + j) * a.g1 * 512 + kb0 * 512;
                // the barrier counts the packed bytes: 64 per row of 128 codes
                const uint32_t bytes = (boxes ? boxes * 32 * 64 : 128 * 64) + 512;
                for (int m = 0; m < 2 && ok; ++m, row += a.I, sf += (int64_t)a.nit * a.g1 * 512) {   // gate, up
                    const int skip = (it & 1) != mine;
                    it += nkb;
                    const uint8_t* f = sf + skip * 512;
                    for (int kb = kb0 + skip; kb < kb1; kb += 2, f += 1024) {
                        if (round && !tc::mbar_wait(empty(s), (round - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                        const uint32_t st = base + st_off + (uint32_t)s * C::kA;
                        tc::mbar_expect_tx(full(s), bytes);
                        if (!boxes) tc::tma_load_2d(st, &tmap_w, kb * 128, row, full(s));
                        else
                            for (int b = 0; b < boxes; ++b) tc::tma_load_2d(st + b * 32 * 128, &tmap_tail, kb * 128, row + 32 * b, full(s));
                        bulk_load(base + sf_off + s * 512, f, 512, full(s));
                        s += 2;
                        if (s >= stages) { s -= stages; ++round; }
                    }
                }
            }
            if (!drain_ring(full(0), stages, s, round, 2, ok)) atomicExch(&s_fail, 1);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            // x's scales stay in tensor memory
            for (int kb = 0; kb < nkb; ++kb) tmem_cp_sf(tmem + C::kSfX + 4 * kb, sf_desc(base + xsf_off + kb * 512));
            int s = 0, par = 0, no = 0;
            bool ok = true;
            for (int item = first; item < items && ok; item += step, ++no) {
                const int buf = no & 1;
                if (no >= 2 && !tc::mbar_wait(acc_empty + 8u * buf, ((no >> 1) - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                tc::tc_fence_after();
                // all of the gate product, then all of up: a change of accumulator costs about 140 clocks, an MMA 57
                for (int m = 0; m < 2 && ok; ++m) {
                    const uint32_t d = tmem + (uint32_t)(buf * C::kAccSet + m * BN);
                    for (int kb = 0; kb < nkb; kb += 2) {
                        const bool two = kb + 1 < nkb;
                        const int s1 = s + 1 == stages ? 0 : s + 1, par1 = s + 1 == stages ? par ^ 1 : par;
                        if (!wait_two(full(s), par, full(s1), par1, two)) { atomicExch(&s_fail, 1); ok = false; break; }
                        const uint32_t sf = tmem + C::kSfW;
                        tmem_cp_sf(sf, sf_desc(base + sf_off + s * 512));
                        if (two) tmem_cp_sf(sf + 4, sf_desc(base + sf_off + s1 * 512));
                        const uint64_t xd = tc::umma_desc_sw128(base + (uint32_t)kb * BN * 128);
                        mma_block<BN>(d, tc::umma_desc_sw128(base + st_off + (uint32_t)s * C::kA), xd, sf, tmem + C::kSfX + 4 * kb, kb > 0);
                        tc::umma_commit(empty(s));
                        if (two) {
                            mma_block<BN>(d, tc::umma_desc_sw128(base + st_off + (uint32_t)s1 * C::kA), xd + BN * 128 / 16, sf + 4, tmem + C::kSfX + 4 * kb + 4, true);
                            tc::umma_commit(empty(s1));
                            s = s1;
                            par = par1;
                        }
                        if (++s == stages) { s = 0; par ^= 1; }
                    }
                }
                tc::umma_commit(acc_full + 8u * buf);
            }
        }
    } else if (warp < 6) {
        const int q = warp & 3;
        const int owner = S == 1 ? 0 : S == 2 ? q >> 1 : q;
        const int slot_q = S == 2 ? q & 1 : 0;            // the owner's slots: its quarters one after the other
        const uint32_t slots = base + recv_off + (uint32_t)(slot_q * (S - 1)) * 2 * BN * 128;
        int no = 0;
        for (int item = first; item < items; item += step, ++no) {
            const int ai = item / a.nit, j = item % a.nit, buf = no & 1, e = R.act[ai];
            const bool done = tc::mbar_wait(acc_full + 8u * buf, (no >> 1) & 1, 4000000000ll);
            tc::tc_fence_after();
            if (!done) atomicExch(&s_fail, 1);
            const bool go = __shfl_sync(0xffffffffu, (done && *(volatile int*)&s_fail == 0) ? 1 : 0, 0) != 0;
            if (!go) break;
            const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * C::kAccSet);
            if (S > 1 && rank != owner) {
                if (!wait_cluster(recv_free + 8u * q, no & 1)) { atomicExch(&s_fail, 1); break; }
                const int src = rank < owner ? rank : rank - 1;
                const uint32_t dst = map_rank(slots + (uint32_t)src * 2 * BN * 128 + lane * 4, owner);
#pragma unroll 1
                for (int t = 0; t < a.T; t += 4) {   // four tokens' gate and up columns; the columns behind T are padding
                    float g[4], u[4];
                    tmem_ld4(acc + t, g);
                    tmem_ld4(acc + BN + t, u);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        st_cluster(dst + (t + i) * 128, g[i]);
                        st_cluster(dst + (BN + t + i) * 128, u[i]);
                    }
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(acc_empty + 8u * buf);
                    arrive_cluster(map_rank(recv_full + 8u * q, owner));
                }
                continue;
            }
            // (the first tile's MMAs are complete, so x's scales have left the slots' place)
            if (S > 1 && no == 0 && lane < S && lane != rank) arrive_cluster(map_rank(recv_free + 8u * q, lane));
            if (S > 1 && !wait_cluster(recv_full + 8u * q, no & 1)) { atomicExch(&s_fail, 1); break; }
            // sums of the S parts in rank order, SwiGLU and the block quantiser: lane = row of I, 32 rows = one block
            const uint32_t mask = R.mask[e];
            float wv = 0.f;
            if (lane < a.T)
                for (int k = 0; k < a.topk; ++k)
                    if (R.sel[lane * kMaxTopk + k] == e) wv = R.wt[lane * kMaxTopk + k];
            const bool real = j * 128 + q * 32 < a.I;
            const int64_t tile = (int64_t)ai * a.nit + j;
            uint8_t* ht = a.h + tile * (BN * 128);
            uint8_t* hs = a.hs + tile * 512;
            const int c16 = q * 2 + (lane >> 4);
#pragma unroll 1
            for (int t = 0; t < a.T; ++t) {
                uint32_t byte = 0, sb = 127;
                if (real && (mask >> t & 1)) {
                    float g, u;
                    tmem_ld1(acc + t, g);
                    tmem_ld1(acc + BN + t, u);
                    tmem_ld_wait();
                    if (S > 1) {
                        const uint32_t at = slots + t * 128 + lane * 4;
                        float gs = 0.f, us = 0.f;
#pragma unroll 1
                        for (int s = 0; s < S; ++s) {
                            float pg = g, pu = u;
                            if (s != rank) {
                                const uint32_t p = at + (uint32_t)(s < rank ? s : s - 1) * 2 * BN * 128;
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(pg) : "r"(p) : "memory");
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(pu) : "r"(p + BN * 128) : "memory");
                            }
                            gs = s ? gs + pg : pg;
                            us = s ? us + pu : pu;
                        }
                        g = gs;
                        u = us;
                    }
                    const float w = __shfl_sync(0xffffffffu, wv, t);
                    const bool nan = g != g || u != u;      // fminf and fmaxf drop a NaN: put it back
                    g = fminf(g, a.limit);
                    u = fminf(fmaxf(u, -a.limit), a.limit);
                    const float hv = nan ? __uint_as_float(0x7fc00000u) : g / (1.f + expf(-g)) * u * w;
                    sb = ue8m0_of(__reduce_max_sync(0xffffffffu, abs_bits(hv)), 1e-4f, kInv448);
                    byte = sb == 255u ? 0u : __nv_cvt_float_to_fp8(hv * ue8m0_inv(sb), __NV_SATFINITE, __NV_E4M3);
                }
                ht[t * 128 + ((c16 ^ (t & 7)) << 4) + (lane & 15)] = (uint8_t)byte;
                if (lane == 0) hs[t * 16 + q] = (uint8_t)sb;
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + 8u * buf);
            if (S > 1 && lane < S && lane != rank) arrive_cluster(map_rank(recv_free + 8u * q, lane));
        }
    }
    __syncwarp();
    tc::tc_fence_before();
    if (S > 1) cluster_sync_all(); else __syncthreads();   // no CTA leaves while a peer may still write to it
    if (threadIdx.x == 0 && s_fail && a.status) { a.status[0] = FB_TIMEOUT; a.status[1] = blockIdx.x; a.status[2] = 1000 + BN; a.status[3] = S; }
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, C::kTmem);
    }
}

template <int BN>
struct DownCfg {
    static constexpr int kA = 128 * 128;
    static constexpr int kStage = kA + BN * 128 + 1024;         // weights, h tile, both scale chunks
    static constexpr int kStages = 10;                          // one CTA per SM: 87 KB of weights in flight
    static constexpr int kTmem = 64;                            // BN accumulator columns + 2 x 8 of scales
    static constexpr size_t kSmem = (size_t)kStages * kStage + 1024 + 256;
    static_assert((size_t)BN * 128 * 4 <= (size_t)kStages * kStage && kStages * 16 + 16 <= 256, "smem");
};

template <int BN, typename TO>
__global__ void __launch_bounds__(kDownThreads, 1)
fp4_moe_down_kernel(const __grid_constant__ CUtensorMap tmap_w, const MoeArgs a) {
    using C = DownCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint16_t s_act[kMaxE];
    __shared__ int s_n;
    __shared__ int s_fail;
    const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + C::kStages * C::kStage;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (C::kStages + s); };
    const uint32_t acc_full = bars + 16u * C::kStages, tmem_slot = acc_full + 8u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = a.S, rank = S > 1 ? (int)cluster_rank() : 0;
    const int tile = blockIdx.x / S, d0 = tile * 128, ntd = (a.D + 127) / 128;
    if (threadIdx.x == 0) {
        s_fail = 0;
        for (int s = 0; s < C::kStages; ++s) {
            tc::mbar_init(full(s), 1);
            tc::mbar_init(empty(s), 1);
        }
        tc::mbar_init(acc_full, 1);
        tc::mbar_fence_init();
        tc::prefetch_tmap(&tmap_w);
    }
    pdl_wait();   // everything below reads what kernel 1 wrote
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, C::kTmem);   // behind the wait: the kernel before need not be kernel 1 (another thread on the stream)
        pdl_launch();   // as in kernel 1
    }
    if (warp >= 2) {
        const volatile int* list = a.list;   // (a read-only load might move above the wait)
        const int n = list[0];
        for (int i = threadIdx.x - 64; i < n; i += kDownThreads - 64) s_act[i] = (uint16_t)list[1 + i];
        if (threadIdx.x == 64) s_n = n;
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    const int64_t units = (int64_t)s_n * a.nit;
    const int u0 = (int)(units * rank / S), u1 = (int)(units * (rank + 1) / S);

    if (warp == 0 || warp == 6) {
        if (elect_one()) {   // two producers, every other block each, as in kernel 1
            const int mine = warp == 6;
            int u = u0 + mine, ai = u / a.nit, kb = u - ai * a.nit, s = mine, round = 0;
            bool ok = true;
            for (; u < u1; u += 2) {
                if (round && !tc::mbar_wait(empty(s), (round - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                const uint32_t st = base + (uint32_t)s * C::kStage;
                const int e = s_act[ai];
                tc::mbar_expect_tx(full(s), 128 * 64 + 512 + BN * 128 + 512);
                tc::tma_load_2d(st, &tmap_w, kb * 128, e * a.D + d0, full(s));
                bulk_load(st + C::kA + BN * 128, a.s2 + (((int64_t)e * ntd + tile) * a.nit + kb) * 512, 512, full(s));
                bulk_load(st + C::kA, a.h + (int64_t)u * (BN * 128), BN * 128, full(s));
                bulk_load(st + C::kA + BN * 128 + 512, a.hs + (int64_t)u * 512, 512, full(s));
                kb += 2;
                while (kb >= a.nit) { kb -= a.nit; ++ai; }
                s += 2;
                if (s >= C::kStages) { s -= C::kStages; ++round; }
            }
            if (!drain_ring(full(0), C::kStages, s, round, 2, ok)) atomicExch(&s_fail, 1);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            int s = 0, par = 0;
            for (int u = u0; u < u1; u += 2) {
                const bool two = u + 1 < u1;
                const int s1 = s + 1 == C::kStages ? 0 : s + 1, par1 = s + 1 == C::kStages ? par ^ 1 : par;
                if (!wait_two(full(s), par, full(s1), par1, two)) { atomicExch(&s_fail, 1); break; }
                const uint32_t st = base + (uint32_t)s * C::kStage, st1 = base + (uint32_t)s1 * C::kStage, sf = tmem + 32;
                tmem_cp_sf(sf, sf_desc(st + C::kA + BN * 128));
                tmem_cp_sf(sf + 4, sf_desc(st + C::kA + BN * 128 + 512));
                if (two) {
                    tmem_cp_sf(sf + 8, sf_desc(st1 + C::kA + BN * 128));
                    tmem_cp_sf(sf + 12, sf_desc(st1 + C::kA + BN * 128 + 512));
                }
                mma_block<BN>(tmem, tc::umma_desc_sw128(st), tc::umma_desc_sw128(st + C::kA), sf, sf + 4, u > u0);
                tc::umma_commit(empty(s));
                if (two) {
                    mma_block<BN>(tmem, tc::umma_desc_sw128(st1), tc::umma_desc_sw128(st1 + C::kA), sf + 8, sf + 12, true);
                    tc::umma_commit(empty(s1));
                    s = s1;
                    par = par1;
                }
                if (++s == C::kStages) { s = 0; par ^= 1; }
            }
            tc::umma_commit(acc_full);
        }
    } else if (warp < 6) {
        const int q = warp & 3;
        const bool done = tc::mbar_wait(acc_full, 0, 4000000000ll);
        tc::tc_fence_after();
        if (!done) atomicExch(&s_fail, 1);
        const bool go = __shfl_sync(0xffffffffu, (done && *(volatile int*)&s_fail == 0) ? 1 : 0, 0) != 0;
        if (go) {
            // the stages are drained: the partial tile [BN][128] goes into them (a rank without blocks has none: zeros)
#pragma unroll
            for (int c = 0; c < BN; c += 8) {
                float r[8];
                tc::tmem_ld8(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + (uint32_t)((c + i) * 128 + q * 32 + lane) * 4), "f"(u1 > u0 ? r[i] : 0.f) : "memory");
            }
        }
        tc::tc_fence_before();
    }
    __syncwarp();
    if (S > 1) cluster_sync_all(); else __syncthreads();
    if (warp >= 2) {
        int bad = 0;
        for (int s = 0; s < S; ++s) {
            int f;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(f) : "r"(S > 1 ? map_rank(tc::smem_u32(&s_fail), s) : tc::smem_u32(&s_fail)) : "memory");
            bad |= f;
        }
        const int t = threadIdx.x - 64, l = t & 127;
        TO* out = reinterpret_cast<TO*>(a.out);
        for (int c = rank * 2 + (t >> 7); c < a.T && !bad; c += 2 * S) {
            const uint32_t at = base + (uint32_t)(c * 128 + l) * 4;
            float p[8];   // all ranks' loads in flight, then the sum in rank order
#pragma unroll
            for (int s = 0; s < 8; ++s) p[s] = s < S ? ld_cluster(S > 1 ? map_rank(at, s) : at) : 0.f;
            float sum = p[0];
#pragma unroll
            for (int s = 1; s < 8; ++s) sum += p[s];
            if (d0 + l < a.D) {
                TO* o = out + c * a.ldo + d0 + l;
                if (a.accumulate) sum += to_f32(*o);
                *o = from_f32<TO>(sum);
            }
        }
    }
    __syncwarp();
    if (S > 1) cluster_sync_all(); else __syncthreads();
    if (threadIdx.x == 0 && s_fail && a.status) { a.status[0] = FB_TIMEOUT; a.status[1] = blockIdx.x; a.status[2] = 2000 + BN; a.status[3] = S; }
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, C::kTmem);
    }
}

// Tensor map of 4-bit codes [rows][cols] (cols a multiple of 128), boxes of 128 codes x box_rows in the padded form.
int make_tmap_u4(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows) {
    if (((uintptr_t)base & 31) || cols % 128) return (int)cudaErrorInvalidValue;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {cols / 2};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fp4_encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, base, dims, strides, box, estr);
}

constexpr int kSms = 148;
constexpr size_t kSmemMax = 227 * 1024 - 10 * 1024;   // dynamic part: the routing tables are static

// Clusters of S CTAs that the device holds at once (a cluster stays inside a GPC, and GPCs lose SMs to odd sizes: 33
// clusters of 4 at one CTA per SM, not 37).  A property of the device and of the kernel's resources.
template <typename F>
int resident_clusters(F kernel, int S, int threads, size_t smem, int per_sm, int* cache /* [9] */) {
    if (S == 1) return kSms * per_sm;
    int n = __atomic_load_n(&cache[S], __ATOMIC_RELAXED);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(S * kSms));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)S;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        n = 1;
    }
    __atomic_store_n(&cache[S], n, __ATOMIC_RELAXED);
    return n;
}

template <int BN, typename F>
int pick_up_cluster(F kernel, int g1, int64_t items, int* stages, int* clusters, int* cache) {
    // Clocks of the longest-running cluster, over the cluster sizes whose x blocks leave room for four stages: per 128-column
    // block of a matrix 300 (four MMAs of 57 and a scale copy), or its bytes' share of HBM if more than 119 CTAs stream;
    // per tile about 1500 in the epilogue that the next tile does not hide, and 2000 more for the exchange of a split.
    int best = 0;
    double cost = 0;
    for (int S = 1; S <= 8 && S <= g1; S *= 2) {
        const int nkb = (g1 + S - 1) / S;
        const size_t fixed = up_fixed<BN>(nkb, S);
        if (nkb > UpCfg<BN>::kMaxKb || fixed + 4 * (size_t)UpCfg<BN>::kStage > kSmemMax) continue;
        int n = (int)((kSmemMax - fixed) / UpCfg<BN>::kStage);
        n = n > 12 ? 12 : n;
        const int64_t nc = resident_clusters(kernel, S, kUpThreads, kSmemMax, 1, cache);
        const int64_t active = (items < nc ? items : nc) * S;
        const double block = active * 2.52 > 300 ? active * 2.52 : 300.0;
        const double c = (double)((items + nc - 1) / nc) * (2 * nkb * block + 1500 + (S > 1 ? 2000 : 0));
        if (!best || c < cost) { best = S; cost = c; *stages = n; *clusters = (int)(items < nc ? items : nc); }
    }
    return best;
}

template <int BN, typename TX>
int launch_up(MoeArgs a, const void* w13, cudaStream_t st) {
    CUtensorMap tw, tt;
    int rc = make_tmap_u4(&tw, w13, (uint64_t)a.E * 2 * a.I, (uint64_t)a.g1 * 128, 128);
    if (!rc) rc = make_tmap_u4(&tt, w13, (uint64_t)a.E * 2 * a.I, (uint64_t)a.g1 * 128, 32);
    if (rc) return rc;
    auto k = fp4_moe_up_kernel<BN, TX>;
    static unsigned long long allowed = 0;
    static int resident[9] = {};
    cudaError_t e = fp4_allow_smem(k, kSmemMax, allowed);
    if (e != cudaSuccess) return (int)e;
    int stages = 0, clusters = 0;
    const int64_t pairs = (int64_t)a.T * a.topk, items = (pairs < a.E ? pairs : a.E) * a.nit;
    a.S = pick_up_cluster<BN>(k, a.g1, items, &stages, &clusters, resident);
    if (!a.S) return (int)cudaErrorInvalidValue;
    const size_t smem = up_fixed<BN>((a.g1 + a.S - 1) / a.S, a.S) + (size_t)stages * UpCfg<BN>::kStage;
    return (int)fp4_launch(k, dim3((unsigned)(clusters * a.S)), dim3(kUpThreads), smem, st, a.S, true, tw, tt, a, stages);
}

template <int BN, typename TO>
int launch_down(MoeArgs a, const void* w2, cudaStream_t st) {
    CUtensorMap tw;
    const int rc = make_tmap_u4(&tw, w2, (uint64_t)a.E * a.D, (uint64_t)a.nit * 128, 128);
    if (rc) return rc;
    auto k = fp4_moe_down_kernel<BN, TO>;
    static unsigned long long allowed = 0;
    cudaError_t e = fp4_allow_smem(k, DownCfg<BN>::kSmem, allowed);
    if (e != cudaSuccess) return (int)e;
    const int tiles = (a.D + 127) / 128;
    const int64_t pairs = (int64_t)a.T * a.topk, units = (pairs < a.E ? pairs : a.E) * a.nit;
    // As many K splits as keep all clusters resident at one CTA per SM, with two blocks each at least.  (Two CTAs per SM
    // take turns on the tensor core, which costs a change of accumulator per block: 0.41 us per block and CTA against
    // 0.165 us alone, and the SMs that got only one CTA wait for the others.)
    static int resident[9] = {};
    int S = 1;
    for (int c = 2; c <= 8; ++c)
        if (units >= 2 * c && tiles <= resident_clusters(k, c, kDownThreads, DownCfg<BN>::kSmem, 1, resident)) S = c;
    a.S = S;
    return (int)fp4_launch(k, dim3((unsigned)(tiles * S)), dim3(kDownThreads), DownCfg<BN>::kSmem, st, S, true, tw, a);
}

template <int BN>
int moe_bn(const MoeArgs& a, const void* w13, const void* w2, cudaStream_t st) {
    int rc = a.xdt == kF32 ? launch_up<BN, float>(a, w13, st) : a.xdt == kBf16 ? launch_up<BN, __nv_bfloat16>(a, w13, st)
                                                                              : launch_up<BN, __half>(a, w13, st);
    if (rc) return rc;
    return a.odt == kF32 ? launch_down<BN, float>(a, w2, st) : a.odt == kBf16 ? launch_down<BN, __nv_bfloat16>(a, w2, st)
                                                                             : launch_down<BN, __half>(a, w2, st);
}

}  // namespace

// x [T, D] (dtype xdt, row stride ldx), logits f32 [T, E] (row stride ldl), bias f32 [E] or null; w13 codes / s13 scales of
// [E, 2, I, D] mxfp4 (gate, up), w2 / s2 of [E, D, I]; out [T, D] (dtype odt, row stride ldo; accumulate: added to);
// score 0 sqrt(softplus), 1 sigmoid, 2 softmax; norm: the chosen scores are divided by their sum (all zero stay zero); limit: SwiGLU clamp
// (infinity: none).  T <= 32, E <= 512, topk <= min(E, 32), I % 32 == 0.  work: 4096 + min(E, T topk) ceil(I / 128) (128 BN
// + 512) bytes, BN = 8 up to 8 tokens, 16 up to 16, else 32.  status: four words that a wait that ran out reports to, or null
// for the device's own (fb_fp4_status).
FB_API int fb_fp4_moe(const void* x, int64_t xdt, int64_t ldx, const float* logits, int64_t ldl, const float* bias, const void* w13,
                      const void* s13, const void* w2, const void* s2, void* out, int64_t odt, int64_t ldo, int64_t accumulate,
                      void* work, int64_t T, int64_t E, int64_t topk, int64_t D, int64_t I, int64_t score, int64_t norm, float scale,
                      float limit, int* status, cudaStream_t st) {
    if (T < 1 || T > kMaxTok || E < 1 || E > kMaxE || topk < 1 || topk > kMaxTopk || topk > E || D < 1 || I < 32 || I % 32 || ldx < D ||
        ldo < D || ldl < E || score < 0 || score > 2 || xdt < 0 || xdt > 2 || odt < 0 || odt > 2 || E * 2 * I > 0x7fffff00ll ||
        E * D > 0x7fffff00ll || D > 0x3fffff || (((uintptr_t)w13 | (uintptr_t)w2) & 31) ||
        (((uintptr_t)s13 | (uintptr_t)s2 | (uintptr_t)work) & 15))
        return (int)cudaErrorInvalidValue;
    MoeArgs a = {};
    a.x = x; a.ldx = ldx; a.logits = logits; a.bias = bias; a.ldl = ldl;
    a.s13 = (const uint8_t*)s13; a.s2 = (const uint8_t*)s2; a.out = out; a.ldo = ldo;
    a.scale = scale; a.limit = limit; a.xdt = (int)xdt; a.odt = (int)odt; a.accumulate = accumulate != 0;
    a.T = (int)T; a.E = (int)E; a.topk = (int)topk; a.D = (int)D; a.I = (int)I; a.score = (int)score; a.norm = norm != 0;
    a.g1 = (int)groups(D); a.nit = (int)((I + 127) / 128);
    a.status = status ? status : fp4_status_ptr();
    if (!a.status) return (int)cudaErrorNotSupported;
    // columns of the MMAs: the cost of an MMA does not depend on them, the room that x and h take in shared memory does
    const int64_t pairs = T * topk < E ? T * topk : E;
    a.list = (int*)work;                         // list, scale chunks, operand tiles: all 16-byte aligned
    a.hs = (uint8_t*)work + 4096;
    a.h = a.hs + pairs * a.nit * 512;
    return T <= 8 ? moe_bn<8>(a, w13, w2, st) : T <= 16 ? moe_bn<16>(a, w13, w2, st) : moe_bn<32>(a, w13, w2, st);
}
