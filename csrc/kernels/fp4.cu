// Block-scaled 4-bit matrices: quantiser and expander (formats and layout: fp4_common.cuh).
//
//   mxfp4   s = 2^ceil(log2(max(amax32, 6 * 2^-126) * (1/6)))           code = e2m1(x / s)
//   nvfp4   u = x / ts (one f32 scale ts for the tensor, or none)       s = e4m3(max(amax16(u), 6 * 2^-9) / 6)
//           code = e2m1(u / s), both quotients rounded to f32 first
//
// Both kernels are bound by HBM (2 + 17/32 bytes per bf16 value) but for the quantiser to nvfp4, whose instructions per
// value weigh as much (83 % of the issue slots).  24896 x 4096 in a graph of many: f32 to either format 68 us (6.8 TB/s), bf16 to
// mxfp4 41.3 us (6.2 TB/s), to nvfp4 47 us (5.5 TB/s; 12 us more with scalar products, a division and a rounded reciprocal
// per block), with a tensor scale 52 us; expanded to bf16 42.5 us (6.1 TB/s), to f32 74 us (6.3 TB/s).  A matrix whose base, row
// stride or width is no multiple of eight values goes by element, in all of its tiles: 24896 x 4095 bf16 75 to 85 us and 289 us
// back, f32 110 and 357 us.  A thread owns eight consecutive
// columns (one 16-byte load of 16-bit values, one 4-byte store of codes), a block of 32 (16) columns is four (two)
// lanes, and a warp takes the four rows i, 32 + i, 64 + i, 96 + i of a 128-row tile over 256 columns: four independent
// loads in flight per thread, and the scales of those rows are 16 consecutive bytes of a chunk, so one lane writes them
// in one store where a row-wise warp would scatter single words over half-filled sectors.
//
// x / s with s a power of two is a product with the exact reciprocal.  For an e4m3 scale the quotient has to be the
// correctly rounded one (a bf16 value over a 4-bit scale often lies exactly on the border of two codes, and a product
// with the rounded reciprocal falls to either side): Markstein's correction, q0 = u r, q = q0 + (u - q0 s) r, two FMAs per
// value (two values per instruction) after one approximate reciprocal per block.
#include "fp4_common.cuh"

namespace {

using namespace fp4;

__device__ int g_fp4_status[4];

constexpr int kQThreads = 256;
constexpr int kQCols = 256;   // columns of a warp's pass

// Tile of this CTA: rows (tile * 128 + 8 * sub + warp) + 32 g, columns 256 * ct ...; bt = matrix of the batch.
struct Place { int64_t bt; int64_t row; int64_t tile; int i; int64_t col; };
__device__ __forceinline__ Place place(int64_t rows, int64_t cols) {
    // 32-bit divisions (the grid has fewer than 2^31 blocks): in 64 bits they were half of the kernel's instructions
    const uint32_t nct = (uint32_t)((cols + kQCols - 1) / kQCols), nrt = (uint32_t)((rows + 127) / 128);
    const uint32_t t = blockIdx.x / nct, ct = blockIdx.x - t * nct, sub = t & 3, rt = t >> 2;
    Place p;
    p.bt = rt / nrt;
    p.tile = rt - (uint32_t)p.bt * nrt;
    p.i = (int)(sub * 8 + (threadIdx.x >> 5));
    p.row = p.tile * 128 + p.i;
    p.col = (int64_t)ct * kQCols + (threadIdx.x & 31) * 8;
    return p;
}

// Whether all of this warp's rows and columns exist (the same for the warps of a CTA but for the last row tile).
__device__ __forceinline__ bool whole(const Place& p, int64_t rows, int64_t cols, int vec) {
    return vec && p.row + 96 < rows && (p.col | 255) < cols;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kQThreads)
fp4_quantize_kernel(const T* x, int64_t ld, int64_t bstride, int vec, uint8_t* codes,
                    uint8_t* scales, int64_t rows, int64_t cols, int scaled, float ts, float inv_ts) {
    pdl_wait();
    pdl_launch();
    const Place p = place(rows, cols);
    const int lane = threadIdx.x & 31;
    const int64_t G = groups(cols), cstride = 64 * G;
    const T* xp = x + p.bt * bstride + p.row * ld + p.col;
    uint8_t* cp = codes + (p.bt * rows + p.row) * cstride + p.col / 2;
    uint32_t bytes = 0;   // the scales of this lane's block in the four rows
    if (whole(p, rows, cols, vec)) {
        const int64_t step = 32 * ld, cstep = 32 * cstride;
        if constexpr (sizeof(T) == 2) {
            uint4 raw[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) raw[g] = ld_v4(xp + g * step);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float v[8];
                uint32_t byte, code;
                unpack8<T>(raw[g], v);
                if (FMT == kNvFp4 && scaled) code = quantize8<FMT>(v, true, ts, inv_ts, byte);
                else code = quantize8<FMT>(v, max_bits8_packed<T>(raw[g]), byte);
                *reinterpret_cast<uint32_t*>(cp + g * cstep) = code;
                bytes |= byte << (8 * g);
            }
        } else {
            float v[4][8];
#pragma unroll
            for (int g = 0; g < 4; ++g) load8(xp + g * step, v[g]);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t byte;
                *reinterpret_cast<uint32_t*>(cp + g * cstep) = quantize8<FMT>(v[g], scaled, ts, inv_ts, byte);
                bytes |= byte << (8 * g);
            }
        }
    } else {
        const int n = (int)max((int64_t)0, min((int64_t)8, cols - p.col));
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
            const bool row = p.row + 32 * g < rows;
            float v[8];
            uint32_t byte;
            load8(row && n ? xp + g * 32 * ld : x, row ? n : 0, false, v);
            const uint32_t code = quantize8<FMT>(v, scaled, ts, inv_ts, byte);
            // codes up to the padded row end (64 bytes per group of 128 columns)
            if (row && p.col < 128 * G) *reinterpret_cast<uint32_t*>(cp + g * 32 * cstride) = code;
            if (row && n > 0) bytes |= byte << (8 * g);
        }
    }
    // four neighbouring blocks (16 lanes of mxfp4, 8 of nvfp4) x four rows: fetch the blocks' words, transpose the bytes
    constexpr int kPer = FMT == kMxFp4 ? 4 : 2;
    const int head = lane & ~(4 * kPer - 1);
    uint32_t w[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) w[b] = __shfl_sync(0xffffffffu, bytes, head + b * kPer);
    constexpr int kChunkCols = FMT == kMxFp4 ? 128 : 64;
    if (lane == head && p.col < 128 * G) {
        const uint32_t a01 = __byte_perm(w[0], w[1], 0x5140), a23 = __byte_perm(w[2], w[3], 0x5140);   // rows 0, 1
        const uint32_t b01 = __byte_perm(w[0], w[1], 0x7362), b23 = __byte_perm(w[2], w[3], 0x7362);   // rows 2, 3
        const int64_t C = FMT == kMxFp4 ? G : 2 * G, nrt = (rows + 127) / 128;
        uint8_t* chunk = scales + ((p.bt * nrt + p.tile) * C + p.col / kChunkCols) * 512;
        *reinterpret_cast<uint4*>(chunk + p.i * 16) = make_uint4(__byte_perm(a01, a23, 0x5410), __byte_perm(a01, a23, 0x7632),
                                                                 __byte_perm(b01, b23, 0x5410), __byte_perm(b01, b23, 0x7632));
    }
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kQThreads)
fp4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* out, int64_t ld,
                      int64_t bstride, int vec, int64_t rows, int64_t cols, float ts) {
    // No early start for the kernel behind this one: what is expanded may be its weights, and the decode GEMVs fetch their first
    // weights before their wait (common.cuh).
    pdl_wait();
    const Place p = place(rows, cols);
    if (p.row >= rows || p.col >= cols) return;
    const int64_t G = groups(cols), cstride = 64 * G, nrt = (rows + 127) / 128;
    constexpr int kChunkCols = FMT == kMxFp4 ? 128 : 64;
    const int64_t C = FMT == kMxFp4 ? G : 2 * G;
    const uint4 sw = ld_v4(scales + ((p.bt * nrt + p.tile) * C + p.col / kChunkCols) * 512 + p.i * 16);
    const uint32_t w[4] = {sw.x, sw.y, sw.z, sw.w};
    uint32_t code[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int64_t r = p.row + 32 * g;
        code[g] = r < rows ? *reinterpret_cast<const uint32_t*>(codes + (p.bt * rows + r) * cstride + p.col / 2) : 0u;
    }
    const int shift = FMT == kMxFp4 ? 8 * (int)(p.col / 32 & 3) : 8 * (int)(p.col / 16 & 3);
    const int n = (int)min((int64_t)8, cols - p.col);
    const bool all = whole(p, rows, cols, vec);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int64_t r = p.row + 32 * g;
        const uint32_t byte = w[g] >> shift & 0xffu;
        float s;
        if (FMT == kMxFp4) {
            // 2^(byte - 127): 0 is the subnormal 2^-127, 255 is NaN
            s = byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
        } else {
            const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
            s = __half2float(*reinterpret_cast<const __half*>(&hr));
        }
        float v[8];
        e2m1x8_to_f32(code[g], v);
        mul8(v, s);
        if (ts != 1.f) mul8(v, ts);
        T* o = out + p.bt * bstride + r * ld + p.col;
        if (all) {
            store8(o, v);
        } else if (r < rows) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) o[j] = from_f32<T>(v[j]);
        }
    }
}

int64_t grid_of(int64_t batch, int64_t rows, int64_t cols) {
    return batch * ((rows + 127) / 128) * 4 * ((cols + kQCols - 1) / kQCols);
}

}  // namespace

int* fp4_status_ptr() {
    static int* cached[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    int* p = __atomic_load_n(&cached[dev], __ATOMIC_ACQUIRE);
    if (!p) {
        void* a = nullptr;
        if (cudaGetSymbolAddress(&a, g_fp4_status) != cudaSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        p = (int*)a;
        __atomic_store_n(&cached[dev], p, __ATOMIC_RELEASE);
    }
    return p;
}

// The status words of the current device's 4-bit kernels into host[4]; waits for the stream.  With `clear` they are zeroed if they
// report something: a report that another stream's kernel makes after the copy stays for the next call.
FB_API int fb_fp4_status(int* host, int64_t clear, cudaStream_t st) {
    int* p = fp4_status_ptr();
    if (!p) return (int)cudaErrorNotSupported;
    cudaError_t e = cudaMemcpyAsync(host, p, 16, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && clear && host[0]) {
        e = cudaMemsetAsync(p, 0, 16, st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    return (int)e;
}

int fp4_quantize(const void* x, int64_t dtype, int64_t ld, int64_t bstride, void* codes, void* scales, int64_t batch, int64_t rows,
                 int64_t cols, int64_t fmt, float ts, bool pdl, cudaStream_t st) {
    if (batch < 1 || rows < 1 || cols < 1 || (fmt != kMxFp4 && fmt != kNvFp4) || dtype < 0 || dtype > 2 ||
        ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15))
        return (int)cudaErrorInvalidValue;
    const int64_t grid = grid_of(batch, rows, cols);
    if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    const int scaled = fmt == kNvFp4 && ts != 0.f && ts != 1.f;
    const float inv = scaled ? (float)(1.0 / (double)ts) : 1.f;
    const int vec = rows_of_8(x, ld, bstride, dtype == kF32 ? 4 : 2);
#define FP4_Q(F, D)                                                                                                         \
    (int)fp4_launch(fp4_quantize_kernel<F, Elem<D>::T>, dim3((unsigned)grid), dim3(kQThreads), 0, st, 1, pdl,  \
                    (const Elem<D>::T*)x, ld, bstride, vec, (uint8_t*)codes, (uint8_t*)scales, rows, cols, scaled, ts, inv)
    if (fmt == kMxFp4) return dtype == kF32 ? FP4_Q(kMxFp4, kF32) : dtype == kBf16 ? FP4_Q(kMxFp4, kBf16) : FP4_Q(kMxFp4, kF16);
    return dtype == kF32 ? FP4_Q(kNvFp4, kF32) : dtype == kBf16 ? FP4_Q(kNvFp4, kBf16) : FP4_Q(kNvFp4, kF16);
#undef FP4_Q
}

// x [batch][rows][cols] (element strides bstride, ld, 1; dtype 0 f32, 1 bf16, 2 f16) -> codes, scales (fp4_common.cuh);
// fmt 0 mxfp4, 1 nvfp4; ts: the tensor's scale (nvfp4, 2^-100 .. 2^100; 0: none).
FB_API int fb_fp4_quantize(const void* x, int64_t dtype, int64_t ld, int64_t bstride, void* codes, void* scales, int64_t batch,
                           int64_t rows, int64_t cols, int64_t fmt, float ts, cudaStream_t st) {
    return fp4_quantize(x, dtype, ld, bstride, codes, scales, batch, rows, cols, fmt, ts, true, st);
}

// codes, scales -> out [batch][rows][cols] (element strides bstride, ld, 1).
FB_API int fb_fp4_dequantize(const void* codes, const void* scales, void* out, int64_t dtype, int64_t ld, int64_t bstride,
                             int64_t batch, int64_t rows, int64_t cols, int64_t fmt, float ts, cudaStream_t st) {
    if (batch < 1 || rows < 1 || cols < 1 || (fmt != kMxFp4 && fmt != kNvFp4) || dtype < 0 || dtype > 2 ||
        ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15))
        return (int)cudaErrorInvalidValue;
    const int64_t grid = grid_of(batch, rows, cols);
    if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    const int vec = rows_of_8(out, ld, bstride, dtype == kF32 ? 4 : 2);
    const float t = ts == 0.f ? 1.f : ts;
#define FP4_D(F, D)                                                                                                    \
    (int)fp4_launch(fp4_dequantize_kernel<F, Elem<D>::T>, dim3((unsigned)grid), dim3(kQThreads), 0, st, 1, true, \
                    (const uint8_t*)codes, (const uint8_t*)scales, (Elem<D>::T*)out, ld, bstride, vec, rows, cols, t)
    if (fmt == kMxFp4) return dtype == kF32 ? FP4_D(kMxFp4, kF32) : dtype == kBf16 ? FP4_D(kMxFp4, kBf16) : FP4_D(kMxFp4, kF16);
    return dtype == kF32 ? FP4_D(kNvFp4, kF32) : dtype == kBf16 ? FP4_D(kNvFp4, kBf16) : FP4_D(kNvFp4, kF16);
#undef FP4_D
}
