// Shared by the block-scaled 4-bit operators (fp4.cu, fp4_gemm.cu, fp4_moe.cu).
//
// A 4-bit matrix [rows, cols] is two byte arrays:
//   codes  [rows][64 * G], G = ceil(cols / 128): two e2m1 codes per byte, the even column in the low nibble, zero codes
//          behind the last column.  A row is then a whole number of 64-byte groups, which is what every TMA box here
//          starts at and what the padded 4-bit TMA form asks of a row.
//   scales [ceil(rows / 128)][C][512], C = G (mxfp4: ue8m0 per 32 columns) or 2 G (nvfp4: e4m3 per 16 columns): byte
//          16 i + 4 g + s of a chunk belongs to row 32 g + i of the 128 and to block s of the chunk's four: the shape
//          that one tcgen05.cp (32x128b, broadcast to the four lane quarters) puts into tensor memory for an MMA.
#pragma once
#include <type_traits>

#include "tc_common.cuh"

enum Fp4Fmt : int { kMxFp4 = 0, kNvFp4 = 1 };
enum Fp4Dtype : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

// fb_fp4_quantize (fp4.cu).  pdl: as for fp4_launch below; without, the product behind it starts earlier (60 x 4096 x 4096: 10.4 us for both
// launches, 11.8 with).
int fp4_quantize(const void* x, int64_t dtype, int64_t ld, int64_t bstride, void* codes, void* scales, int64_t batch, int64_t rows,
                 int64_t cols, int64_t fmt, float ts, bool pdl, cudaStream_t st);

// Device words that the bounded waits of these kernels report to (the current device's copy); null if CUDA refuses.
int* fp4_status_ptr();

// Launch with an optional cluster of `cluster` CTAs along x and, with `pdl`, programmatic serialisation: the kernel's start-up
// runs beside the end of the kernel before it.  The rules that make that safe here:
//   * a kernel touches no memory before its griddepcontrol.wait, so completion is transitive along the stream; the one
//     exception is the product behind its own quantiser, which reads the weights: the quantiser lets it start after its own
//     wait, when everything before the quantiser is complete;
//   * the expander lets nothing start early, because its output may be the weights of a kernel that reads them before its wait;
//   * a kernel that waits for another holds no tensor memory that the other may still ask for: tensor memory is taken
//     after the wait.  Of the kernel before nothing is presumed, not even behind a launch of the same call: two host threads
//     may share a stream, and many a kernel lets its dependents start before it has taken its own.
template <typename... KArgs, typename... Args>
inline cudaError_t fp4_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, bool pdl,
                              Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    if (e != cudaSuccess) (void)cudaGetLastError();   // reported to this caller, not to the next launch
    return e;
}

// cuTensorMapEncodeTiled, 2-D, no interleave, zero fill.
inline int fp4_encode_tmap(CUtensorMap* map, CUtensorMapDataType type, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                           const cuuint32_t* box, const cuuint32_t* estr, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || !p)
            return (int)cudaErrorNotSupported;
        fn = (EncodeFn)p;
    }
    const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// cudaFuncSetAttribute once per kernel and device.
template <typename F>
inline cudaError_t fp4_allow_smem(F kernel, size_t bytes, unsigned long long& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (__atomic_load_n(&done, __ATOMIC_RELAXED) >> dev & 1)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) __atomic_fetch_or(&done, 1ull << dev, __ATOMIC_RELAXED);
    return e;
}

namespace fp4 {

constexpr float kInv6 = 1.f / 6.f;
constexpr float kInv448 = 1.f / 448.f;

__host__ __device__ __forceinline__ int64_t groups(int64_t cols) { return (cols + 127) / 128; }

__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* gsrc, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_dst), "l"(gsrc), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Shared-memory descriptor of a 512-byte scale chunk (no swizzle, 8-row groups 128 bytes apart).
__device__ __forceinline__ uint64_t sf_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void tmem_cp_sf(uint32_t taddr, uint64_t sdesc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// One lane of a converged warp.  The lanes that feed TMA and the tensor core are chosen this way and not by `lane == 0`: the
// compiler then knows that the branch has one thread and keeps descriptors and addresses in uniform registers.  Measured
// on a loop of four small MMAs, a scale copy, a commit and a wait: 252 clocks instead of 524.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

// End of a producer of a ring of stages: its copies have landed, whatever the other warps came to (after a wait that ran out the CTA
// would end with copies on their way into its shared memory; without one they have landed long before).  full0: the first stage's
// barrier; s, round: where the next block would go.  step 1: one producer.  step 2: two that take every other block; this one
// has issued (round stages + s) / 2 blocks, and of these only the last stages / 2 are looked at: a stage further back may be the
// other one's by now, whose phases would be taken for its own.  That one alone is looked at after a failure, when nothing more is
// issued and a wait in vain costs its budget.
__device__ __forceinline__ bool drain_ring(uint32_t full0, int stages, int s, int round, int step, bool ok) {
    const int issued = (round * stages + s) / step;
    for (int i = 0; i < issued && i < (stages + (ok ? 0 : step - 1)) / step; ++i) {
        s -= step;
        if (s < 0) { s += stages; --round; }
        if (!tc::mbar_wait(full0 + 8u * s, round & 1)) return false;
    }
    return true;
}

// Tiled TMA store of a box in shared memory (clipped at the tensor's ends) and its bulk groups (per thread).
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t smem_src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_src) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }

// ---- clusters ------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t smem_addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// ---- codes -----------------------------------------------------------------------------------------
// Eight f32 -> eight e2m1 codes (round to nearest, ties to even, saturating), value j in nibble j.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t d;
    asm("{\n .reg .b8 b0, b1, b2, b3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        " mov.b32 %0, {b0, b1, b2, b3};\n}"
        : "=r"(d) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}
// Eight codes -> eight f32 (exact).
__device__ __forceinline__ void e2m1x8_to_f32(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// |x| as an integer: NaN > inf > every number, so a maximum of these keeps what a float maximum would drop.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

// Power-of-two scale exponent byte (ue8m0) of a block: 2^ceil(log2(amax * (1 / top))), amax floored.  255 (NaN) for a
// block that holds an infinity or a NaN.
__device__ __forceinline__ uint32_t ue8m0_of(uint32_t amax_bits, float floor, float inv_top) {
    if (amax_bits >= kInfBits) return 255u;
    const uint32_t b = __float_as_uint(__fmul_rn(fmaxf(__uint_as_float(amax_bits), floor), inv_top));
    return (b >> 23) + ((b & 0x7fffffu) != 0u);
}
// 1 / 2^(e - 127) for e in 1..253
__device__ __forceinline__ float ue8m0_inv(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// Two f32 in a register pair: the products and sums below take both in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ void mul8(float (&v)[8], float f) {
    const uint64_t ff = pair(f, f);
#pragma unroll
    for (int j = 0; j < 8; j += 2) unpair(mul2(pair(v[j], v[j + 1]), ff), v[j], v[j + 1]);
}

// u / s rounded to nearest, from r = rn(1 / s): Markstein's correction of the product u r.  For an s of four significant bits
// (an e4m3 number) an r that is off by 2^-22 will do: the residual u - q0 s is exact, so q0 + residual r is off by less than
// 2^-20 of a step before its rounding, and u / s is never nearer than 1/32 of a step to the middle of two f32 (u and the
// middle times s are both multiples of 2^-28 of u's binade, and they differ: the middle's 25 bits, times an odd s, are no f32).
__device__ __forceinline__ float div_by(float u, float s, float r) {
    const float q0 = __fmul_rn(u, r);
    return __fmaf_rn(__fmaf_rn(-q0, s, u), r, q0);
}
__device__ __forceinline__ void div8_by(float (&v)[8], float s, float r) {
    const uint64_t ns = pair(-s, -s), rr = pair(r, r);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t u = pair(v[j], v[j + 1]), q0 = mul2(u, rr);
        unpair(fma2(fma2(q0, ns, u), rr, q0), v[j], v[j + 1]);
    }
}

// Eight consecutive values of a row (m: the largest of their |.| as integer, the values divided by the tensor scale already)
// -> their codes (value j in nibble j) and the scale byte of their block, which is this lane and its neighbours (four
// lanes of mxfp4, two of nvfp4; whole warps call).
template <int FMT>
__device__ __forceinline__ uint32_t quantize8(float (&v)[8], uint32_t m, uint32_t& byte) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    if (FMT == kMxFp4) m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (FMT == kMxFp4) {
        byte = ue8m0_of(m, 6.f * 1.17549435e-38f, kInv6);
        const float inv = ue8m0_inv(min(byte, 253u));
        mul8(v, inv);
    } else {
        byte = m >= kInfBits ? 0x7fu
                             : (uint32_t)__nv_cvt_float_to_fp8(div_by(fmaxf(__uint_as_float(m), 6.f / 512.f), 6.f, kInv6), __NV_SATFINITE, __NV_E4M3);
        const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
        const float s = __half2float(*reinterpret_cast<const __half*>(&hr));
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
        div8_by(v, s, r);   // correctly rounded although r is not: see div_by
    }
    return m >= kInfBits ? 0u : e2m1x8(v);   // a block that is not finite: NaN scale, zero codes
}

// max(|a|, |b|) that keeps a NaN (as the largest integer).
__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
// Largest |.| of eight values as an integer that orders NaN > infinity > numbers.
__device__ __forceinline__ uint32_t max_bits8(const float (&v)[8]) {
    float m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = max_abs_nan(v[2 * j], v[2 * j + 1]);
    return __float_as_uint(max_abs_nan(max_abs_nan(m[0], m[1]), max_abs_nan(m[2], m[3])));
}

// The same with the values as they are loaded; scaled: nvfp4 with a tensor scale ts.
template <int FMT>
__device__ __forceinline__ uint32_t quantize8(float (&v)[8], bool scaled, float ts, float inv_ts, uint32_t& byte) {
    if (FMT == kNvFp4 && scaled) {
        div8_by(v, ts, inv_ts);
    }
    return quantize8<FMT>(v, max_bits8(v), byte);
}

// Whether rows of a matrix can be read and written eight values at a time.
inline bool rows_of_8(const void* p, int64_t ld, int64_t bstride, int esz) {
    return (uintptr_t)p % (8 * esz) == 0 && ld % 8 == 0 && bstride % 8 == 0;
}

// ---- values of the three element types -----------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<kF32> { using T = float; };
template <> struct Elem<kBf16> { using T = __nv_bfloat16; };
template <> struct Elem<kF16> { using T = __half; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Largest |.| of eight 16-bit values as they are in memory (two per word), in the integer form of max_bits8.
template <typename T>
__device__ __forceinline__ uint32_t max_bits8_packed(const uint4& a) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        auto h = [](uint32_t w) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)); };
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h(a.x), h(a.y)), __hmax2_nan(h(a.z), h(a.w)));
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
        return max(w << 16, w & 0xffff0000u);
    } else {
        auto h = [](uint32_t w) { return __habs2(*reinterpret_cast<const __half2*>(&w)); };
        const __half2 m = __hmax2_nan(__hmax2_nan(h(a.x), h(a.y)), __hmax2_nan(h(a.z), h(a.w)));
        return max(abs_bits(__low2float(m)), abs_bits(__high2float(m)));
    }
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& a, float (&v)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            v[2 * i] = bf16lo(w[i]);
            v[2 * i + 1] = bf16hi(w[i]);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
// (volatile, and no read-only loads: what these read may still be written by the kernel before while this one starts)
__device__ __forceinline__ uint4 ld_v4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ float ld_f32(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
// p[0 .. 7] -> f32, all of them there; p is aligned to the eight values (16 bytes, f32 32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
    } else {
        unpack8<T>(ld_v4(p), v);
    }
}
// The first n of them (the others read 0); vec: p is aligned as above.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
    if (vec && n >= 8) {
        load8(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}
// Eight values as they are in memory.
template <typename T> struct Raw8 {
    uint4 w;
    __device__ __forceinline__ void load(const T* p) { w = ld_v4(p); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const { unpack8<T>(w, v); }
    __device__ __forceinline__ uint32_t max_bits() const { return max_bits8_packed<T>(w); }
};
template <> struct Raw8<float> {
    float f[8];
    __device__ __forceinline__ void load(const float* p) { load8(p, f); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = f[j];
    }
    __device__ __forceinline__ uint32_t max_bits() const { return max_bits8(f); }
};
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// Eight values to p (aligned as for load8).
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                     "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

}  // namespace fp4
