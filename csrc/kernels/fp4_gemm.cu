// Product of two block-scaled 4-bit matrices on the 5th-generation tensor cores:
//
//   out[m, n] = alpha * sum_k X[m, k] W[n, k],   X, W = e2m1 codes times block scales (fp4_common.cuh)
//
// tcgen05.mma kind::mxf4 (ue8m0 per 32, two scales per K = 64 step) or kind::mxf4nvf4 (e4m3 per 16, four per step):
// both operands stay packed in shared memory (128 bytes = 256 values per row, 128-byte swizzle) and the hardware
// applies the scales, which tcgen05.cp moves from shared to tensor memory.  Nothing is expanded anywhere.
//
// The operand on the 128 lanes of the accumulator is called P, the other one Q (BN columns).  Many rows: P = X, so a
// thread of the epilogue holds neighbouring outputs of one row.  Few rows (one tile of Q holds all of X): P = W, the
// weights fill the lanes whatever the number of rows, and the K axis is split over a cluster of S CTAs whose partial
// tiles are summed in rank order through distributed shared memory: no workspace, no atomics, the same bits every run.
//
// Bounds (times in graphs of many calls).  Few rows: the weights' bytes from HBM; 1 x 5120 x 129280 mxfp4 59 us (5.9 TB/s), 1 x 8192 x
// 5120 8.8 us (3.4 for the bytes), 16 x 4096 x 24896 nvfp4 14.8 us with its quantiser (8.9 for the bytes: the rest is the latency of
// two launches and of the first tiles).  Many rows: the tensor cores and the operands' way from L2; 8192 x 8192 x 8192 mxfp4 192 us
// (5.7 PFLOP/s, twenty calls after a pause), nvfp4 217 us, 8192 x 4096 x 24896 nvfp4 404 us, where repeated calls run into the
// power cap (about 1.55 GHz).
//
// Warps: 0 producer (TMA boxes of both operands, bulk copies of the scale chunks), 1 MMA issuer, 2..9 epilogue (two per
// lane quarter).  Without a split the CTAs are persistent and walk the tiles; the accumulator is handed to the epilogue
// and back through two barriers.  Every wait has a clock budget; on expiry the status words say so, the tile is not
// stored, the copies in flight are waited for and the tensor memory is released.
#include "fp4_common.cuh"

namespace {

using namespace fp4;

constexpr int kBK = 256;          // values per stage row (128 bytes)
constexpr int kGThreads = 320;
constexpr int kEpi = 256;         // epilogue threads: two warps per lane quarter
constexpr int kQxBlocks = 16;     // QX: blocks of X that a CTA holds

template <int FMT, int BN, bool SWAP, bool QX>
struct GemmCfg {
    static constexpr int kChunks = FMT == kMxFp4 ? 2 : 4;              // scale chunks of a stage per 128 rows
    static constexpr int kQAtoms = (BN + 127) / 128;
    static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
    static constexpr int kSfa = 512 * kChunks, kSfb = kSfa * kQAtoms;
    static constexpr int kXBlock = kBBytes + kSfb;   // QX: a block of X (256 columns of K) lives outside the stages
    static constexpr int kStageBytes = (kABytes + kSfa + (QX ? 0 : kXBlock) + 1023) / 1024 * 1024;
    // P = X: each epilogue warp stages its rows of the output in two buffers of 32 rows x 128 bytes
    static constexpr int kStaging = SWAP ? 0 : (kEpi / 32) * 2 * 4096;
    static constexpr int kBudget = BN <= 32 && !QX ? 112 * 1024 : 227 * 1024;  // up to 32 columns: two CTAs per SM (1x129280x5120
                                                                        // mxfp4 61.2 us, 62.9 with one of twice the stages)
    static constexpr int kBars = 512;
    static constexpr int kXRoom = QX ? kQxBlocks * kXBlock : 0;
    static constexpr int kFit = (kBudget - kBars - kStaging - kXRoom) / kStageBytes;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr int kSfCols = 4 * kChunks * (1 + kQAtoms);        // tensor memory columns of a stage's scales
    static constexpr int kAcc = BN < 32 ? 32 : BN;
    static constexpr int kNeed = kAcc + 2 * kSfCols;
    static constexpr int kTmem = kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kXRoom + kStaging + kBars;
    static_assert(kStages >= 3 && kStages * 16 + 32 <= kBars, "stages");
    static_assert((size_t)BN * 128 * 4 <= (size_t)kStages * kStageBytes, "the partial tile reuses the stages");
};

template <int FMT>
__host__ __device__ constexpr uint32_t fp4_idesc(int N, int sf) {
    // A, B: e2m1 (1); scale type ue8m0 (1) or ue4m3 (0); M = 128; sf: scale byte of the 32-bit word, both operands
    return ((uint32_t)sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((FMT == kMxFp4 ? 1u : 0u) << 23) |
           ((128u >> 4) << 24) | ((uint32_t)sf << 29);
}
template <int FMT>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    if constexpr (FMT == kMxFp4)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
}

struct GemmArgs {
    const uint8_t *sfp, *sfq;
    const void* x;            // QX: the rows to quantise (row stride ldx, element type xdt; tensor scale xts if scaled)
    int64_t ldx;
    float xts, xinv;
    int xdt, scaled;
    void* out;
    int64_t ldo;
    int64_t P, Q, K;
    float alpha;
    int dtype, vec, tail, tiles_p, tiles_q, splits;   // vec: TMA can address out; tail: its rows end inside a 16-byte unit
    int behind;               // the kernel before this one is the quantiser of X, and everything before that is complete
    int* status;
};

// P = W (few rows of X): lane = output column, a warp's store is 32 neighbouring outputs of one row.
template <typename T, int BN>
__device__ __forceinline__ void store_columns(const GemmArgs& a, uint32_t tmem, int warp, int lane, int64_t p0, int64_t q0) {
    // warp w of 0..7: lane quarter w & 3, column half w >> 2
    const int quarter = warp & 3;
    const int64_t p = p0 + quarter * 32 + lane;
    constexpr int kHalf = BN >= 32 ? BN / 2 : BN;
    if (BN < 32 && warp >= 4) return;
    const int c0 = (warp >> 2) * kHalf;
#pragma unroll 1
    for (int c = c0; c < c0 + kHalf && q0 + c < a.Q; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, r);
        tmem_ld_wait();
        if (p >= a.P) continue;
        const int n = (int)min((int64_t)16, a.Q - (q0 + c));
        T* out = reinterpret_cast<T*>(a.out) + (q0 + c) * a.ldo + p;
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n) out[j * a.ldo] = from_f32<T>(__uint_as_float(r[j]) * a.alpha);
    }
}

// P = X: a lane holds a row's outputs side by side.  They go through two buffers of 32 rows x ROW bytes of this warp
// (16-byte units swizzled as in TMA's 128- or 64-byte mode) and leave as TMA stores, which the tensor core does not wait
// for: the accumulator is given back as soon as it is read.  Rows that TMA cannot address (base or row stride not a
// multiple of 16 bytes) leave as stores of 32 neighbouring outputs, and so does a tile in which rows end inside a 16-byte unit: TMA
// clips a box at whole units, and what is behind a row's end is not the output's.  (Decided per tile: a test per buffer, or the
// last unit alone by element, cost all tiles 1.3 to 4 % of 1024 x 4096 x 24896.)
template <typename T, int BN, int ROW, bool PAIR = false>
__device__ __forceinline__ void store_rows(const GemmArgs& a, const CUtensorMap* tmap_o, uint32_t tmem, uint32_t buf0, int warp, int lane,
                                           int64_t p0, int64_t q0, bool vec, uint32_t acc_empty, int& turn) {
    constexpr int kCols = ROW / (int)sizeof(T), kChunks = BN / 2 / kCols;   // columns of a buffer, buffers of this warp's half
    auto unit = [](int row, int u) { return (uint32_t)(row * ROW + ((u ^ (ROW == 128 ? row & 7 : row >> 1 & 3)) << 4)); };
    static_assert(kChunks >= 1, "a warp's half is a buffer at least");
    const int quarter = warp & 3, c0 = (warp >> 2) * (BN / 2);
    const int64_t row0 = p0 + quarter * 32;
#pragma unroll 1
    for (int ch = 0; ch < kChunks; ++ch, turn ^= 1) {   // the buffers take turns, across tiles too
        const uint32_t buf = buf0 + (uint32_t)turn * (32 * ROW);
        const int64_t q = q0 + c0 + ch * kCols;
        if (lane == 0) bulk_wait_read<1>();      // the store before the last has left this buffer
        __syncwarp();
        uint32_t r[kCols];
#pragma unroll
        for (int c = 0; c < kCols; c += 16) tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c0 + ch * kCols + c), *reinterpret_cast<uint32_t(*)[16]>(r + c));
        tmem_ld_wait();
        if (ch == kChunks - 1) {
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(acc_empty) : "memory");
                else mbar_arrive(acc_empty);
            }
        }
#pragma unroll
        for (int u = 0; u < ROW / 16; ++u) {     // 16-byte units
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(__uint_as_float(r[u * 4 + i]) * a.alpha);
                else w[i] = pack2<T>(__uint_as_float(r[u * 8 + 2 * i]) * a.alpha, __uint_as_float(r[u * 8 + 2 * i + 1]) * a.alpha);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + unit(lane, u)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        if (vec) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                if (q < a.Q && row0 < a.P) tma_store_2d(tmap_o, (int)q, (int)row0, buf);
                bulk_commit();
            }
        } else {
            __syncwarp();
            const int rows = (int)min((int64_t)32, a.P - row0);
#pragma unroll 1
            for (int i = 0; i < rows; ++i) {
                T* out = reinterpret_cast<T*>(a.out) + (row0 + i) * a.ldo + q;
#pragma unroll
                for (int h = 0; h < kCols; h += 32) {
                    const int c = h + lane % (kCols < 32 ? kCols : 32), byte = c * (int)sizeof(T);
                    T v;
                    const uint32_t at = buf + unit(i, byte >> 4) + (byte & 15);
                    if constexpr (sizeof(T) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
                    else { uint16_t u; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(at) : "memory"); v = *reinterpret_cast<T*>(&u); }
                    if (q + c < a.Q) out[c] = v;
                }
            }
            __syncwarp();
            if (lane == 0) bulk_commit();   // an empty group: the wait above counts buffers
        }
    }
}

template <typename T, bool SWAP, int BN>
__device__ __forceinline__ void store_reduced(const GemmArgs& a, uint32_t part, int t, int rank, int64_t p0, int64_t q0) {
    // part: this CTA's partial tile [BN][128] f32 in shared memory; ranks own the column groups of 128 lanes in turn
    T* out = reinterpret_cast<T*>(a.out);
    const int S = a.splits, lane = t & 127;
    for (int c = rank * 2 + (t >> 7); c < BN; c += 2 * S) {
        if (q0 + c >= a.Q) break;
        float v[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) v[s] = s < S ? ld_cluster(map_rank(part + (uint32_t)(c * 128 + lane) * 4, s)) : 0.f;
        float sum = v[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) sum += v[s];
        const int64_t p = p0 + lane, q = q0 + c;
        if (p < a.P) out[SWAP ? q * a.ldo + p : p * a.ldo + q] = from_f32<T>(sum * a.alpha);
    }
}

// The K range of X (kb0 .. kb1 in blocks of 256 columns) quantised into operand form: per block [BN][128 bytes] swizzled
// codes, then the scale chunks.  Columns behind K count as zeros (their scales have to be numbers).
template <int FMT, typename C>
__device__ __forceinline__ void quantize_x(const GemmArgs& a, uint8_t* room, int t, int kb0, int kb1, uint32_t x_full, int lane) {
    pdl_wait();
    const int units = (kb1 - kb0) * 32;                    // of eight columns
    const int esz = a.xdt == kF32 ? 4 : 2;
    const bool vec = (uintptr_t)a.x % (8 * esz) == 0 && a.ldx % 8 == 0;
#pragma unroll 1
    for (int64_t m = 0; m < a.Q; ++m) {
#pragma unroll 1
        for (int c0 = 0; c0 < units; c0 += kEpi) {
            const int c = c0 + t;
            const int64_t col = (int64_t)kb0 * kBK + 8 * c;
            const int n = c < units ? (int)max((int64_t)0, min((int64_t)8, a.K - col)) : 0;
            const int64_t at = m * a.ldx + (n ? col : 0);
            float v[8];
            if (a.xdt == kBf16) load8(reinterpret_cast<const __nv_bfloat16*>(a.x) + at, n, vec, v);
            else if (a.xdt == kF16) load8(reinterpret_cast<const __half*>(a.x) + at, n, vec, v);
            else load8(reinterpret_cast<const float*>(a.x) + at, n, vec, v);
            uint32_t byte;
            const uint32_t code = quantize8<FMT>(v, a.scaled != 0, a.xts, a.xinv, byte);
            if (c < units) {
                uint8_t* blk = room + (c >> 5) * C::kXBlock;
                const int u = c & 31;                      // 4 bytes of codes each
                *reinterpret_cast<uint32_t*>(blk + m * 128 + (((u >> 2) ^ (int)(m & 7)) << 4) + (u & 3) * 4) = code;
                constexpr int kPer = FMT == kMxFp4 ? 4 : 2;
                const int b = u / kPer;                    // block of the 256 columns
                if (u % kPer == 0) blk[C::kBBytes + (b >> 2) * 512 + m * 16 + (b & 3)] = (uint8_t)byte;
            }
        }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(x_full);
}

template <int FMT, int BN, bool SWAP, bool QX>
__global__ void __launch_bounds__(kGThreads, BN <= 32 && !QX ? 2 : 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                const __grid_constant__ CUtensorMap tmap_o, const GemmArgs a) {
    using C = GemmCfg<FMT, BN, SWAP, QX>;
    // no static shared memory: the swizzled tiles start on 1024 bytes without padding (three stages and the staging buffers
    // of the widest tile fill all but 768 bytes)
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = tc::smem_u32(smem_raw);
    const uint32_t xroom = base + C::kStages * C::kStageBytes;   // (the SWAP forms have no staging buffers, the others no X room)
    const uint32_t staging = xroom, bars = xroom + C::kXRoom + C::kStaging;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (C::kStages + s); };
    const uint32_t acc_full = bars + 16u * C::kStages, acc_empty = acc_full + 8u, tmem_slot = acc_full + 16u, x_full = acc_full + 24u;
    int& s_fail = *reinterpret_cast<int*>(smem_raw + (acc_full + 20u - base));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = a.splits, rank = S > 1 ? (int)cluster_rank() : 0;
    const int64_t G = groups(a.K);
    const int64_t Cch = FMT == kMxFp4 ? G : 2 * G;
    const int nkb_all = (int)((G + 1) / 2);
    const int kb0 = (int)((int64_t)nkb_all * rank / S), kb1 = (int)((int64_t)nkb_all * (rank + 1) / S);
    // the last stage of K: 64-column MMA steps that hold columns, bytes of scale chunks per 128 rows
    constexpr uint32_t kFull = 512 * C::kChunks;
    const int tail_steps = (int)((a.K - (int64_t)(nkb_all - 1) * kBK + 63) / 64);
    const uint32_t tail_sf = 512 * (uint32_t)(Cch - (int64_t)(nkb_all - 1) * C::kChunks);
    const int n_tiles = a.tiles_p * a.tiles_q;
    const int first = S > 1 ? blockIdx.x / S : blockIdx.x, step = S > 1 ? n_tiles : gridDim.x;
    // tiles in bands of kBand along P, so that the CTAs in flight share operand tiles through L2
    constexpr int kBand = 8;
    auto tile_at = [&](int t, int64_t& p0, int64_t& q0) {
        const int band = t / (kBand * a.tiles_q), in = t - band * kBand * a.tiles_q;
        const int h = min(kBand, a.tiles_p - band * kBand);
        p0 = (int64_t)(band * kBand + in % h) * 128;
        q0 = (int64_t)(in / h) * BN;
    };

    if (threadIdx.x == 0) {
        s_fail = (base & 1023u) != 0;   // (never: then nothing is stored and the status says so)
        for (int s = 0; s < C::kStages; ++s) {
            tc::mbar_init(full(s), 1);
            tc::mbar_init(empty(s), 1);
        }
        tc::mbar_init(acc_full, 1);
        tc::mbar_init(acc_empty, kEpi / 32);
        if (QX) tc::mbar_init(x_full, kEpi / 32);
        tc::mbar_fence_init();
        tc::prefetch_tmap(&tmap_p);
        tc::prefetch_tmap(&tmap_q);
        if (!SWAP) tc::prefetch_tmap(&tmap_o);
    }
    __syncthreads();
    // Tensor memory, for every warp but the producer.  It is taken behind the wait: whatever kernel is before this one in
    // the stream (another host thread may have put one between the quantiser and this launch) may still ask for its own.
    uint32_t tmem = 0;
    if (warp >= 1) {
        if constexpr (QX) {
            if (warp >= 2) quantize_x<FMT, C>(a, smem_raw + (xroom - base), threadIdx.x - 64, kb0, kb1, x_full, lane);
        }
        if (warp == 1) {
            pdl_wait();
            tc::tmem_alloc(tmem_slot, C::kTmem);
            pdl_launch();
        }
        tc::tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(kGThreads - 32) : "memory");
        tc::tc_fence_after();
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    }
    const uint32_t a_off = 0, b_off = C::kABytes, sfa_off = b_off + (QX ? 0 : C::kBBytes), sfb_off = sfa_off + C::kSfa;

    if (warp == 0) {
        if (elect_one()) {
            // One thread's dependent instructions are what a stage costs here: addresses are advanced, not computed, and only the
            // last stage of K looks at how much of it there is.
            const int q_rowtiles = (int)((a.Q + 127) / 128);
            const uint32_t pbytes = C::kABytes + kFull, qbytes = QX ? 0u : C::kBBytes;
            auto load_p = [&](int s, int kb, int p0, const uint8_t* f, uint32_t sf) {
                tc::tma_load_2d(base + s * C::kStageBytes + a_off, &tmap_p, kb * 128, p0, full(s));
                bulk_load(base + s * C::kStageBytes + sfa_off, f, sf, full(s));
            };
            auto load_q = [&](int s, int kb, int q0, const uint8_t* f, uint32_t sf, int at) {
                if (QX) return;
                tc::tma_load_2d(base + s * C::kStageBytes + b_off, &tmap_q, kb * 128, q0, full(s));
                bulk_load(base + s * C::kStageBytes + sfb_off, f, sf, full(s));
                if (C::kQAtoms > 1 && at > 1) bulk_load(base + s * C::kStageBytes + sfb_off + C::kSfa, f + Cch * 512, sf, full(s));
            };
            int s = 0, round = 0;
            bool ok = true;
            for (int t = first; t < n_tiles && ok; t += step) {
                int64_t p0, q0;
                tile_at(t, p0, q0);
                const int at = min(C::kQAtoms, q_rowtiles - (int)(q0 / 128));
                const uint8_t* fp = a.sfp + ((p0 / 128) * Cch + (int64_t)kb0 * C::kChunks) * 512;
                const uint8_t* fq = QX ? nullptr : a.sfq + ((q0 / 128) * Cch + (int64_t)kb0 * C::kChunks) * 512;
                const uint32_t qat = QX ? 0u : (uint32_t)at;
                int kb = kb0;
                if (t == first && !a.behind) pdl_wait();
                if (t == first && a.behind) {
                    // X is written by the kernel before this one: only W (P when swapped) may be read before the wait
                    const int ahead = SWAP ? min(C::kStages, kb1 - kb0) : 0;
                    for (int i = 0; i < ahead; ++i) {
                        const uint32_t sf = kb0 + i == nkb_all - 1 ? tail_sf : kFull;
                        tc::mbar_expect_tx(full(i), C::kABytes + qbytes + sf * (1 + qat));
                        load_p(i, kb0 + i, (int)p0, fp + i * kFull, sf);
                    }
                    pdl_wait();
                    for (int i = 0; i < ahead; ++i) load_q(i, kb0 + i, (int)q0, fq + i * kFull, kb0 + i == nkb_all - 1 ? tail_sf : kFull, at);
                    kb += ahead;
                    fp += ahead * kFull;
                    fq += ahead * kFull;
                    s = ahead;
                    if (s == C::kStages) { s = 0; round = 1; }
                }
                for (; kb < kb1; ++kb, fp += kFull, fq += kFull) {
                    if (round && !tc::mbar_wait(empty(s), (round - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                    const uint32_t sf = kb == nkb_all - 1 ? tail_sf : kFull;
                    tc::mbar_expect_tx(full(s), kb == nkb_all - 1 ? C::kABytes + qbytes + sf * (1 + qat) : pbytes + qbytes + kFull * qat);
                    load_p(s, kb, (int)p0, fp, sf);
                    load_q(s, kb, (int)q0, fq, sf, at);
                    if (++s == C::kStages) { s = 0; ++round; }
                }
            }
            if (!drain_ring(full(0), C::kStages, s, round, 1, ok)) atomicExch(&s_fail, 1);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            int s = 0, par = 0, flip = 0, tile_no = 0;
            bool ok = true;
            if (QX && !tc::mbar_wait(x_full, 0)) { atomicExch(&s_fail, 1); ok = false; }
            for (int t = first; t < n_tiles && ok; t += step, ++tile_no) {
                if (tile_no && !tc::mbar_wait(acc_empty, (tile_no - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                tc::tc_fence_after();
                uint32_t xb = xroom;   // QX: this stage's block of X
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!tc::mbar_wait(full(s), par)) { atomicExch(&s_fail, 1); ok = false; break; }
                    tc::tc_fence_after();
                    const uint32_t st = base + s * C::kStageBytes;
                    const uint32_t sfa_t = tmem + C::kAcc + (uint32_t)flip, sfb_t = sfa_t + 4 * C::kChunks;
                    flip ^= C::kSfCols;
                    const uint32_t sfa_s = st + sfa_off, sfb_s = QX ? xb + C::kBBytes : st + sfb_off;
                    const uint64_t ad = tc::umma_desc_sw128(st + a_off), bd = tc::umma_desc_sw128(QX ? xb : st + b_off);
                    auto scales = [&](int c) {   // word c of all atoms side by side: 4 columns per 128 rows
                        tmem_cp_sf(sfa_t + 4 * c, sf_desc(sfa_s + 512 * c));
#pragma unroll
                        for (int at = 0; at < C::kQAtoms; ++at) tmem_cp_sf(sfb_t + 4 * (c * C::kQAtoms + at), sf_desc(sfb_s + at * C::kSfa + 512 * c));
                    };
                    auto mma = [&](int k) {
                        const int c = FMT == kMxFp4 ? k / 2 : k;
                        umma_fp4<FMT>(tmem, ad + 2u * k, bd + 2u * k, fp4_idesc<FMT>(BN, FMT == kMxFp4 ? 2 * (k & 1) : 0), sfa_t + 4 * c,
                                      sfb_t + 4 * c * C::kQAtoms, (kb > kb0 || k) ? 1u : 0u);
                    };
                    if (kb < nkb_all - 1 || tail_steps == 4) {
#pragma unroll
                        for (int c = 0; c < C::kChunks; ++c) scales(c);
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma(k);
                    } else {
                        for (int c = 0; c < (FMT == kMxFp4 ? (tail_steps + 1) / 2 : tail_steps); ++c) scales(c);
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            if (k < tail_steps) mma(k);
                    }
                    tc::umma_commit(empty(s));
                    if (++s == C::kStages) { s = 0; par ^= 1; }
                    xb += C::kXBlock;
                }
                tc::umma_commit(acc_full);
            }
        }
    } else {
        const int w = warp - 2;
        // warps 2..9: TMEM lane quarter = warp & 3
        const int quarter_warp = (warp & 3) | (w >= 4 ? 4 : 0);
        int tile_no = 0, turn = 0;
        for (int t = first; t < n_tiles; t += step, ++tile_no) {
            int64_t p0, q0;
            tile_at(t, p0, q0);
            const bool done = tc::mbar_wait(acc_full, tile_no & 1, 4000000000ll);
            tc::tc_fence_after();
            if (!done) atomicExch(&s_fail, 1);
            const bool go = __shfl_sync(0xffffffffu, (done && *(volatile int*)&s_fail == 0) ? 1 : 0, 0) != 0;
            if (S > 1) {
                // the stages are drained (every MMA of this CTA is complete): the partial tile goes into them
                if (go) {
                    const int quarter = quarter_warp & 3;
                    constexpr int kHalf = BN >= 32 ? BN / 2 : BN;
                    if (BN >= 32 || quarter_warp < 4) {
                        const int c0 = (quarter_warp >> 2) * kHalf;
#pragma unroll 1
                        for (int c = c0; c < c0 + kHalf; c += 16) {
                            uint32_t r[16];
                            tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, r);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + (uint32_t)((c + j) * 128 + quarter * 32 + lane) * 4), "r"(r[j]) : "memory");
                        }
                    }
                }
            } else if (go) {
                if constexpr (SWAP) {
                    if (a.dtype == kBf16) store_columns<__nv_bfloat16, BN>(a, tmem, quarter_warp, lane, p0, q0);
                    else if (a.dtype == kF16) store_columns<__half, BN>(a, tmem, quarter_warp, lane, p0, q0);
                    else store_columns<float, BN>(a, tmem, quarter_warp, lane, p0, q0);
                } else {
                    const uint32_t buf = staging + (uint32_t)w * 8192;
                    const bool vec = a.vec && (!a.tail || q0 + BN <= a.Q);
                    if (a.dtype == kBf16) store_rows<__nv_bfloat16, BN, 128>(a, &tmap_o, tmem, buf, quarter_warp, lane, p0, q0, vec, acc_empty, turn);
                    else if (a.dtype == kF16) store_rows<__half, BN, 128>(a, &tmap_o, tmem, buf, quarter_warp, lane, p0, q0, vec, acc_empty, turn);
                    else store_rows<float, BN, 128>(a, &tmap_o, tmem, buf, quarter_warp, lane, p0, q0, vec, acc_empty, turn);
                    continue;   // (store_rows gave the accumulator back)
                }
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);   // also after a failed wait
            if (!go) break;
        }
        if (!SWAP && S == 1 && lane == 0) bulk_wait<0>();
    }
    __syncwarp();
    tc::tc_fence_before();
    if (S > 1) {
        // s_fail of every CTA is final and its partial tile is visible to the cluster
        cluster_sync_all();
        if (warp >= 2) {
            int64_t p0, q0;
            tile_at(first, p0, q0);
            int bad = 0;
            for (int s = 0; s < S; ++s) {
                int f;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(f) : "r"(map_rank(tc::smem_u32(&s_fail), s)) : "memory");
                bad |= f;
            }
            if (!bad) {
                const int t = threadIdx.x - 64;
                if (a.dtype == kBf16) store_reduced<__nv_bfloat16, SWAP, BN>(a, base, t, rank, p0, q0);
                else if (a.dtype == kF16) store_reduced<__half, SWAP, BN>(a, base, t, rank, p0, q0);
                else store_reduced<float, SWAP, BN>(a, base, t, rank, p0, q0);
            }
        }
        cluster_sync_all();   // nobody leaves while a peer still reads its tile
    } else {
        __syncthreads();
    }
    if (threadIdx.x == 0 && s_fail && a.status) { a.status[0] = FB_TIMEOUT; a.status[1] = blockIdx.x; a.status[2] = BN; a.status[3] = S; }
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, C::kTmem);
    }
}

// ---- pairs of CTAs -----------------------------------------------------------------------------------------------
// One tile of 256 rows of X x 256 rows of W per cluster of two CTAs (tcgen05.mma cta_group::2): each CTA holds 128 rows of
// either operand and the accumulator of its 128 rows of X; the MMA, issued by rank 0, reads both CTAs' halves of W.  A
// CTA then fetches 32 KB of codes per 256 columns of K where the single-CTA tile of 128 x 256 fetches 48 KB, and the
// fabric between L2 and the SMs (about 64 bytes per clock and SM) was what that one waited for.
// All copies of a stage, both CTAs', complete on rank 0's barrier (TMA with cta_group::2 may signal the pair's other CTA):
// a first form in which rank 1 passed its completions on took 1370 clocks a stage instead of about 700.
template <int FMT>
struct PairCfg {
    static constexpr int kChunks = FMT == kMxFp4 ? 2 : 4;
    static constexpr int kA = 128 * 128, kB = 128 * 128;
    static constexpr int kSfa = 512 * kChunks, kSfb = 2 * kSfa;          // scales: this CTA's rows of X, all 256 rows of W
    static constexpr int kStageBytes = kA + kB + kSfa + kSfb;
    static constexpr int kStaging = (kEpi / 32) * 2 * 2048, kBars = 512;   // 64-byte rows: room for a fifth stage
    static constexpr int kStages = 5;
    static constexpr int kSfCols = 4 * kChunks * 3;
    static constexpr int kAcc = 256, kTmem = 512;
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kStaging + kBars;
    static_assert(kStageBytes % 1024 == 0 && kSmem <= 227 * 1024 && kAcc + 2 * kSfCols <= kTmem, "sizes");
};
// TMA box into this CTA's shared memory, completion on a barrier of either CTA of the pair (shared::cluster address).
__device__ __forceinline__ void tma_load_pair(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int FMT>
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    if constexpr (FMT == kMxFp4)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
}
__device__ __forceinline__ void cp_sf_pair(uint32_t taddr, uint64_t sdesc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
// Arrives on the barrier at this offset in both CTAs when the MMAs issued so far are complete.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

template <int FMT>
__global__ void __launch_bounds__(kGThreads, 1)
fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                     const __grid_constant__ CUtensorMap tmap_sp, const __grid_constant__ CUtensorMap tmap_sq,
                     const __grid_constant__ CUtensorMap tmap_o, const GemmArgs a) {
    using C = PairCfg<FMT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = tc::smem_u32(smem_raw);
    const uint32_t staging = base + C::kStages * C::kStageBytes, bars = staging + C::kStaging;
    auto full = [&](int s) { return bars + 8u * s; };                     // (rank 0's alone is used)
    auto empty = [&](int s) { return bars + 8u * (C::kStages + s); };
    const uint32_t acc_full = bars + 16u * C::kStages, acc_empty = acc_full + 8u, tmem_slot = acc_full + 16u;
    int& s_fail = *reinterpret_cast<int*>(smem_raw + (acc_full + 20u - base));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int64_t G = groups(a.K), Cch = FMT == kMxFp4 ? G : 2 * G;
    const int nkb = (int)((G + 1) / 2);
    const int tail_steps = (int)((a.K - (int64_t)(nkb - 1) * kBK + 63) / 64), tail_chunks = FMT == kMxFp4 ? (tail_steps + 1) / 2 : tail_steps;
    const int n_tiles = a.tiles_p * a.tiles_q, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    constexpr int kBand = 4;   // bands of tiles along P, so that the pairs in flight share operand tiles through L2
    auto tile_at = [&](int t, int64_t& p0, int64_t& q0) {
        const int band = t / (kBand * a.tiles_q), in = t - band * kBand * a.tiles_q;
        const int h = min(kBand, a.tiles_p - band * kBand);
        p0 = (int64_t)(band * kBand + in % h) * 256;
        q0 = (int64_t)(in / h) * 256;
    };
    if (threadIdx.x == 0) {
        s_fail = (base & 1023u) != 0;
        for (int s = 0; s < C::kStages; ++s) {
            tc::mbar_init(full(s), 1);
            tc::mbar_init(empty(s), 1);
        }
        tc::mbar_init(acc_full, 1);
        tc::mbar_init(acc_empty, 2 * kEpi / 32);
        tc::mbar_fence_init();
        tc::prefetch_tmap(&tmap_p);
        tc::prefetch_tmap(&tmap_q);
        tc::prefetch_tmap(&tmap_o);
    }
    if (warp == 1) {
        pdl_wait();   // before the tensor memory, as above
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "n"(C::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        pdl_launch();
    }
    tc::tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc::tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    constexpr uint32_t b_off = C::kA, sfa_off = C::kA + C::kB, sfb_off = sfa_off + C::kSfa;

    if (warp == 0) {
        if (elect_one()) {
            pdl_wait();
            int s = 0, round = 0;
            bool ok = true;
            const uint32_t lead = map_rank(full(0), 0);
            for (int t = first; t < n_tiles && ok; t += step) {
                int64_t p0, q0;
                tile_at(t, p0, q0);
                // rows of 512 bytes in the scale maps: chunks; what lies behind a matrix's or a row's end reads something finite
                // or zero and meets no stored output
                int sp = (int)((p0 / 128 + rank) * Cch), sq = (int)(q0 / 128 * Cch), sq1 = sq + (int)Cch;
                for (int kb = 0; kb < nkb; ++kb) {
                    if (round && !tc::mbar_wait(empty(s), (round - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                    const uint32_t st = base + s * C::kStageBytes, bar = lead + 8u * s;
                    if (rank == 0) tc::mbar_expect_tx(full(s), 2 * C::kStageBytes);
                    tma_load_pair(st, &tmap_p, kb * 128, (int)p0 + 128 * rank, bar);
                    tma_load_pair(st + b_off, &tmap_q, kb * 128, (int)q0 + 128 * rank, bar);
                    tma_load_pair(st + sfa_off, &tmap_sp, 0, sp, bar);
                    tma_load_pair(st + sfb_off, &tmap_sq, 0, sq, bar);
                    tma_load_pair(st + sfb_off + C::kSfa, &tmap_sq, 0, sq1, bar);
                    sp += C::kChunks;
                    sq += C::kChunks;
                    sq1 += C::kChunks;
                    if (++s == C::kStages) { s = 0; ++round; }
                }
            }
            // (rank 0's barriers count both CTAs' copies, and rank 1 stays until rank 0 is through)
            if (rank == 0 && !drain_ring(full(0), C::kStages, s, round, 1, ok)) atomicExch(&s_fail, 1);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            int s = 0, par = 0;
            bool ok = true;
            if (rank == 0) {
                int it = 0, tile_no = 0;
                for (int t = first; t < n_tiles && ok; t += step, ++tile_no) {
                    if (tile_no && !tc::mbar_wait(acc_empty, (tile_no - 1) & 1)) { atomicExch(&s_fail, 1); ok = false; break; }
                    tc::tc_fence_after();
                    for (int kb = 0; kb < nkb; ++kb, ++it) {
                        if (!tc::mbar_wait(full(s), par)) { atomicExch(&s_fail, 1); ok = false; break; }
                        tc::tc_fence_after();
                        const uint32_t st = base + s * C::kStageBytes;
                        const uint32_t sfa_t = tmem + C::kAcc + (uint32_t)(it & 1) * C::kSfCols, sfb_t = sfa_t + 4 * C::kChunks;
                        const int steps = kb == nkb - 1 ? tail_steps : 4, nch = kb == nkb - 1 ? tail_chunks : C::kChunks;
                        auto scales = [&](int c) {
                            if (c >= nch) return;
                            cp_sf_pair(sfa_t + 4 * c, sf_desc(st + sfa_off + 512 * c));
                            cp_sf_pair(sfb_t + 8 * c, sf_desc(st + sfb_off + 512 * c));
                            cp_sf_pair(sfb_t + 8 * c + 4, sf_desc(st + sfb_off + C::kSfa + 512 * c));
                        };
                        const uint64_t ad = tc::umma_desc_sw128(st), bd = tc::umma_desc_sw128(st + b_off);
                        // the copies of a word's scales go one word ahead of its MMAs: they run beside the MMAs before them
                        scales(0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (k >= steps) break;
                            const int c = FMT == kMxFp4 ? k / 2 : k;
                            if (FMT == kNvFp4 || k % 2 == 0) scales(c + 1);
                            // M = 256 of the pair: the field of fp4_idesc holds M = 128
                            umma_pair<FMT>(tmem, ad + 2u * k, bd + 2u * k, fp4_idesc<FMT>(256, FMT == kMxFp4 ? 2 * (k & 1) : 0) + ((128u >> 4) << 24),
                                           sfa_t + 4 * c, sfb_t + 8 * c, (kb | k) ? 1u : 0u);
                        }
                        commit_pair(empty(s));
                        if (++s == C::kStages) { s = 0; par ^= 1; }
                    }
                    commit_pair(acc_full);
                }
            }
        }
    } else {
        const int w = warp - 2, quarter_warp = (warp & 3) | (w >= 4 ? 4 : 0);
        const uint32_t peer_empty = map_rank(acc_empty, 0);               // (rank 0's, for both)
        int tile_no = 0, turn = 0;
        for (int t = first; t < n_tiles; t += step, ++tile_no) {
            int64_t p0, q0;
            tile_at(t, p0, q0);
            const bool done = tc::mbar_wait(acc_full, tile_no & 1, 4000000000ll);
            tc::tc_fence_after();
            if (!done) atomicExch(&s_fail, 1);
            const bool go = __shfl_sync(0xffffffffu, (done && *(volatile int*)&s_fail == 0) ? 1 : 0, 0) != 0;
            if (!go) break;
            const uint32_t buf = staging + (uint32_t)w * 4096;
            const bool vec = a.vec && (!a.tail || q0 + 256 <= a.Q);
            const int64_t pr = p0 + 128 * rank;
            if (a.dtype == kBf16) store_rows<__nv_bfloat16, 256, 64, true>(a, &tmap_o, tmem, buf, quarter_warp, lane, pr, q0, vec, peer_empty, turn);
            else if (a.dtype == kF16) store_rows<__half, 256, 64, true>(a, &tmap_o, tmem, buf, quarter_warp, lane, pr, q0, vec, peer_empty, turn);
            else store_rows<float, 256, 64, true>(a, &tmap_o, tmem, buf, quarter_warp, lane, pr, q0, vec, peer_empty, turn);
        }
        if (lane == 0) bulk_wait<0>();
    }
    __syncwarp();
    tc::tc_fence_before();
    cluster_sync_all();   // no CTA leaves while the pair's MMAs, commits or arrivals may still reach it
    if (threadIdx.x == 0 && s_fail && a.status) { a.status[0] = FB_TIMEOUT; a.status[1] = blockIdx.x; a.status[2] = 3000; a.status[3] = rank; }
    if (warp == 1) {
        tc::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kTmem) : "memory");
    }
}

// Output [rows, cols] in boxes of 32 rows x row_bytes (128 or 64), swizzled.
int make_tmap_out(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols, uint64_t ld, int dtype, int row_bytes) {
    static_assert(kF32 == 0 && kBf16 == 1 && kF16 == 2, "the order of the table below");
    const CUtensorMapDataType types[3] = {CU_TENSOR_MAP_DATA_TYPE_FLOAT32, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16};
    const uint64_t esz = dtype == kF32 ? 4 : 2;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {ld * esz};
    cuuint32_t box[2] = {(cuuint32_t)(row_bytes / esz), 32};
    cuuint32_t estr[2] = {1, 1};
    return fp4_encode_tmap(map, types[dtype], base, dims, strides, box, estr, row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// Scale chunks as rows of 128 words, in boxes of `box_rows`.
int make_tmap_scales(CUtensorMap* map, const void* base, uint64_t chunks, uint32_t box_rows) {
    cuuint64_t dims[2] = {128, chunks};
    cuuint64_t strides[1] = {512};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fp4_encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, dims, strides, box, estr, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int FMT, int BN, bool SWAP, bool QX = false>
int launch_gemm(const GemmArgs& a, const void* pc, const void* qc, int grid, cudaStream_t st) {
    using C = GemmCfg<FMT, BN, SWAP, QX>;
    CUtensorMap tp, tq, to;
    const uint64_t bytes = (uint64_t)(64 * groups(a.K));
    // the row end (a multiple of 64 bytes) lies inside a 128-byte box of the last stage: what is behind it reads zero
    int rc = fb_make_tmap_2d(&tp, pc, (uint64_t)a.P, bytes, 128, 128, 1);
    tq = to = tp;   // (QX has no operand Q in memory; `to` is not used by P = W or an output that TMA cannot address)
    if (!rc && !QX) rc = fb_make_tmap_2d(&tq, qc, (uint64_t)a.Q, bytes, BN, 128, 1);
    if (!rc && !SWAP && a.vec) rc = make_tmap_out(&to, a.out, (uint64_t)a.P, (uint64_t)a.Q, (uint64_t)a.ldo, a.dtype, 128);
    if (rc) return rc;
    auto k = fp4_gemm_kernel<FMT, BN, SWAP, QX>;
    static unsigned long long allowed = 0;
    cudaError_t e = fp4_allow_smem(k, C::kSmem, allowed);
    if (e != cudaSuccess) return (int)e;
    return (int)fp4_launch(k, dim3((unsigned)grid), dim3(kGThreads), C::kSmem, st, a.splits, true, tp, tq, to, a);
}

// Clusters of 1 .. 8 CTAs that fit the device at one CTA per SM (measured: a cluster stays inside a GPC).
constexpr int kResident[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
constexpr int kNotTaken = -1;     // X is not quantised inside the product at these sizes
constexpr int kQxRows = 16;       // rows times blocks of 256 columns per CTA up to which it is

template <int FMT>
int launch_pair(GemmArgs a, const void* pc, const void* qc, cudaStream_t st) {
    using C = PairCfg<FMT>;
    CUtensorMap tp, tq, tsp, tsq, to;
    const uint64_t bytes = (uint64_t)(64 * groups(a.K)), cch = (uint64_t)(FMT == kMxFp4 ? 1 : 2) * groups(a.K);
    int rc = fb_make_tmap_2d(&tp, pc, (uint64_t)a.P, bytes, 128, 128, 1);
    if (!rc) rc = fb_make_tmap_2d(&tq, qc, (uint64_t)a.Q, bytes, 128, 128, 1);
    if (!rc) rc = make_tmap_scales(&tsp, a.sfp, (uint64_t)((a.P + 127) / 128) * cch, C::kChunks);
    if (!rc) rc = make_tmap_scales(&tsq, a.sfq, (uint64_t)((a.Q + 127) / 128) * cch, C::kChunks);
    to = tp;   // (not used by an output that TMA cannot address)
    if (!rc && a.vec) rc = make_tmap_out(&to, a.out, (uint64_t)a.P, (uint64_t)a.Q, (uint64_t)a.ldo, a.dtype, 64);
    if (rc) return rc;
    auto k = fp4_gemm_pair_kernel<FMT>;
    static unsigned long long allowed = 0;
    cudaError_t e = fp4_allow_smem(k, C::kSmem, allowed);
    if (e != cudaSuccess) return (int)e;
    const int tiles = a.tiles_p * a.tiles_q, pairs = 74;
    return (int)fp4_launch(k, dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs))), dim3(kGThreads), C::kSmem, st, 2, true, tp, tq, tsp, tsq, to, a);
}

template <int FMT>
int gemm_fmt(GemmArgs a, const void* xc, const uint8_t* xs, const void* wc, const uint8_t* ws, int64_t M, int64_t N, cudaStream_t st) {
    const int sms = 148;
    const int nkb = (int)((groups(a.K) + 1) / 2);
    if (M <= 128) {
        // weights on the lanes; as many K splits as fill the SMs, with at least two stages each
        const int bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
        a.P = N; a.Q = M; a.sfp = ws; a.sfq = xs;
        a.tiles_p = (int)((N + 127) / 128);
        a.tiles_q = 1;
        // K split by the clocks of the longest-running CTA, as below: a stage takes its MMAs and scale copies or, with many
        // CTAs, its share of HBM (17.4 KB of weights at 3450 bytes per clock)
        const double mma = bn <= 32 ? 350 : bn == 64 ? 400 : 470;
        double cost = 0;
        int S = 1;
        for (int c = 1; c <= 8; ++c) {
            if (c > 1 && (a.tiles_p > kResident[c] || nkb < 2 * c)) continue;
            const int64_t active = (int64_t)(a.tiles_p < kResident[c] ? a.tiles_p : kResident[c]) * c;
            const double stage = active * 5.05 > mma ? active * 5.05 : mma;
            const double t = (double)((a.tiles_p + kResident[c] - 1) / kResident[c]) * (((nkb + c - 1) / c) * stage + 1500) + (c > 1 ? 3000 : 0);
            if (cost == 0 || t < cost) { cost = t; S = c; }
        }
        a.splits = S;
        const int slots = bn <= 32 && !a.x ? 2 * sms : sms;
        const int grid = S > 1 ? a.tiles_p * S : (a.tiles_p < slots ? a.tiles_p : slots);
        if (a.x) {
            // Rows that are quantised on the way: with few values per CTA its idle epilogue warps do it while the first weights
            // arrive, and the quantiser's own launch goes.
            if (bn > 16 || (nkb + S - 1) / S > kQxBlocks || M * ((nkb + S - 1) / S) > kQxRows) return kNotTaken;
            return launch_gemm<FMT, 16, true, true>(a, wc, nullptr, grid, st);
        }
        switch (bn) {
            case 16: return launch_gemm<FMT, 16, true>(a, wc, xc, grid, st);
            case 32: return launch_gemm<FMT, 32, true>(a, wc, xc, grid, st);
            case 64: return launch_gemm<FMT, 64, true>(a, wc, xc, grid, st);
            default: return launch_gemm<FMT, 128, true>(a, wc, xc, grid, st);
        }
    }
    if (a.x) return kNotTaken;
    a.P = M; a.Q = N; a.sfp = xs; a.sfq = ws;
    a.tiles_p = (int)((M + 127) / 128);
    // Tile and K split by the clocks of the longest-running CTA: a stage (256 columns of K) takes about 850 on 256
    // output columns and 560 on 128 (the operands' way from L2), 600 in a pair, a tile about 1500 at its ends that the next one does
    // not hide, an exchange between split CTAs 3000.  Clusters of a split stay resident.
    double cost = 0;
    bool wide = true;
    int S = 1;
    for (int w = 0; w < 2; ++w) {
        const int64_t tiles = (int64_t)a.tiles_p * ((N + (w ? 255 : 127)) / (w ? 256 : 128));
        for (int l = 0; l < 4; ++l) {
            const int s = 1 << l;
            if (l && (tiles > kResident[s] || nkb < 2 * s)) break;
            const double c = (double)((tiles + sms - 1) / sms) * ((double)((nkb + s - 1) / s) * (w ? 850 : 560) + 1500) + (s > 1 ? 3000 : 0);
            if (cost == 0 || c < cost) { cost = c; wide = w; S = s; }
        }
    }
    const int64_t pair_p = (M + 255) / 256, pair_q = (N + 255) / 256, pair_tiles = pair_p * pair_q;
    if (pair_tiles > 0x3fffffff) return (int)cudaErrorInvalidValue;
    if ((double)((pair_tiles + 73) / 74) * ((double)nkb * 600 + 1700) < cost) {
        a.tiles_p = (int)pair_p;
        a.tiles_q = (int)pair_q;
        a.splits = 1;
        return launch_pair<FMT>(a, xc, wc, st);
    }
    a.tiles_q = (int)((N + (wide ? 255 : 127)) / (wide ? 256 : 128));
    const int64_t tiles = (int64_t)a.tiles_p * a.tiles_q;
    if (tiles > 0x3fffffff) return (int)cudaErrorInvalidValue;
    a.splits = S;
    const int grid = S > 1 ? (int)tiles * S : (int)(tiles < sms ? tiles : sms);
    if (wide) return launch_gemm<FMT, 256, false>(a, xc, wc, grid, st);
    return launch_gemm<FMT, 128, false>(a, xc, wc, grid, st);
}

}  // namespace

static int fp4_matmul(const void* xc, const void* xs, const void* wc, const void* ws, int64_t M, int64_t N, int64_t fmt, GemmArgs a,
                      int* status, cudaStream_t st) {
    if (M < 1 || N < 1 || a.K < 1 || M > 0x7fffff00ll || N > 0x7fffff00ll || a.K > 0x3fffff00ll || a.ldo < N || a.dtype < 0 || a.dtype > 2 ||
        (fmt != kMxFp4 && fmt != kNvFp4) || (((uintptr_t)xc | (uintptr_t)xs | (uintptr_t)wc | (uintptr_t)ws) & 15))
        return (int)cudaErrorInvalidValue;
    const int esz = a.dtype == kF32 ? 4 : 2;
    a.vec = ((uintptr_t)a.out & 15) == 0 && a.ldo * esz % 16 == 0;
    a.tail = N * esz % 16 != 0;
    a.status = status ? status : fp4_status_ptr();
    if (!a.status) return (int)cudaErrorNotSupported;
    return fmt == kMxFp4 ? gemm_fmt<kMxFp4>(a, xc, (const uint8_t*)xs, wc, (const uint8_t*)ws, M, N, st)
                         : gemm_fmt<kNvFp4>(a, xc, (const uint8_t*)xs, wc, (const uint8_t*)ws, M, N, st);
}

// out[M, N] (row stride ldo, dtype 0 f32, 1 bf16, 2 f16) = alpha * X W^T of two 4-bit matrices of one format with K columns.
// status: four words that a wait that ran out reports to, or null for the device's own (fb_fp4_status).
FB_API int fb_fp4_matmul(const void* xc, const void* xs, const void* wc, const void* ws, void* out, int64_t dtype, int64_t ldo,
                         int64_t M, int64_t N, int64_t K, int64_t fmt, float alpha, int* status, cudaStream_t st) {
    GemmArgs a = {};
    a.out = out; a.ldo = ldo; a.K = K; a.alpha = alpha; a.dtype = (int)dtype;
    return fp4_matmul(xc, xs, wc, ws, M, N, fmt, a, status, st);
}

// The same with the rows of x [M, K] (element type xdt, row stride ldx; nvfp4: tensor scale xts or 0) quantised first: inside the
// product for few values, else by fb_fp4_quantize into `work`: codes [M][64 ceil(K / 128)], then (at the next multiple of
// 512) the scale chunks; the product's prologue and its first weight tiles overlap that launch.  (One row of up to 4096
// columns never needs `work`.)
FB_API int fb_fp4_linear(const void* x, int64_t xdt, int64_t ldx, void* work, const void* wc, const void* ws, void* out,
                         int64_t dtype, int64_t ldo, int64_t M, int64_t N, int64_t K, int64_t fmt, float xts, float alpha,
                         int* status, cudaStream_t st) {
    if (M < 1 || K < 1 || xdt < 0 || xdt > 2 || ldx < K || ((uintptr_t)work & 15)) return (int)cudaErrorInvalidValue;
    GemmArgs a = {};
    a.out = out; a.ldo = ldo; a.K = K; a.alpha = alpha; a.dtype = (int)dtype;
    a.x = x; a.ldx = ldx; a.xdt = (int)xdt;
    a.scaled = fmt == kNvFp4 && xts != 0.f && xts != 1.f;
    a.xts = xts;
    a.xinv = a.scaled ? (float)(1.0 / (double)xts) : 1.f;
    int rc = fp4_matmul(nullptr, nullptr, wc, ws, M, N, fmt, a, status, st);
    if (rc != kNotTaken) return rc;
    if (!work) return (int)cudaErrorInvalidValue;
    uint8_t* codes = (uint8_t*)work;
    uint8_t* scales = codes + (M * 64 * groups(K) + 511) / 512 * 512;
    rc = fp4_quantize(x, xdt, ldx, 0, codes, scales, 1, M, K, fmt, xts, false, st);
    if (rc) return rc;
    a.x = nullptr;
    a.behind = 1;
    return fp4_matmul(codes, scales, wc, ws, M, N, fmt, a, status, st);
}
