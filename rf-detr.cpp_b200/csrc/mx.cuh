// Microscaled 4-bit operands (MXFP4) and the operators on them: quantisation, product, the norms
// around a transformer block (which can write such an operand), and attention over packed
// sequences.
//
// A matrix [rows][k] is held as
//   codes   [rows][ld bytes], E2M1, two to a byte (the even column in the low nibble); a row holds
//           ceil(k / 32) * 16 bytes, zeros behind column k
//   scales  one E8M0 byte 2^(e - 127) for 32 values, in the order the tensor cores take them:
//           tiles of 128 rows x 4 blocks (512 bytes), the tiles of 128 rows side by side along k;
//           row r, block b of a tile at byte (r % 32) * 16 + (r / 32) * 4 + b.  Rows and blocks that
//           fill up the last tiles are zeros.
// The scale of a block is 2^(floor(log2 max|x|) - 2): the block's largest value lies in [4, 8) of it
// and E2M1 reaches 6 (the conversion of the OCP Microscaling Formats specification, v1.0).  A block
// with an infinity or a NaN has scale 0xFF (NaN) and codes 0.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "rfdetr_b200.h"

namespace rfb {

// element types by their GGUF ids
enum : int { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 30 };
enum : int { NORM_NONE = 0, NORM_LAYER = 1, NORM_RMS = 2 };

inline bool mx_type_ok(int t) { return t == MX_F32 || t == MX_F16 || t == MX_BF16; }
inline int mx_type_size(int t) { return t == MX_F32 ? 4 : 2; }
inline bool ptr_aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
// a code matrix as TMA and the vector stores take it
inline bool mx_codes_ok(const void* p, int ld, int k) {
    return p && ptr_aligned(p, 16) && ld % 16 == 0 && (long long)ld >= ((long long)k + 31) / 32 * 16;
}

// cuTensorMapEncodeTiled of the driver, or nullptr
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// The error word of device `dev`, the current one: 0 until a kernel's wait runs out (sm100.cuh).
cudaError_t op_error_word(int dev, int** word);

cudaError_t mx_quantize(const void* src, int type, int ld, int rows, int k, uint8_t* codes, int ldc, uint8_t* scales,
                        cudaStream_t st);
cudaError_t mx_dequantize(const uint8_t* codes, int ldc, const uint8_t* scales, int rows, int k, void* dst, int type,
                          int ld, cudaStream_t st);
cudaError_t mx_gemm(const uint8_t* a, int lda, const uint8_t* a_scales, const uint8_t* b, int ldb,
                    const uint8_t* b_scales, int M, int N, int K, int act, const float* bias, void* out, int out_type,
                    int ldo, cudaStream_t st);
cudaError_t block_norm(const rfdetr_b200_block_norm& p, cudaStream_t st);
cudaError_t attention_packed(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv, void* o, int ldo,
                             int type, const int32_t* cu_seqlens, int n_seqs, int tokens, int max_len, int heads,
                             int kv_heads, int head_dim, int causal, float scale, cudaStream_t st);

// ---- device helpers ----------------------------------------------------------

// byte of row r's scale of block b; kt = tiles along k
__host__ __device__ __forceinline__ size_t mx_scale_at(int r, int b, int kt) {
    return ((size_t)(r >> 7) * kt + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

// Threads that write the zeros behind the last row of an operand whose rows end inside a tile.
inline long long mx_pad_threads(int kt) { return 32ll * kt; }

#ifdef __CUDACC__

// The operators' kernels are launched while the stream's previous kernel still runs (where that lets them): each lets
// the next start once its own CTAs have, and touches memory only behind the wait for all work before it.  What earlier work
// may have written changes while such a kernel is there already, so it is read by plain loads: neither __ldg nor __restrict__,
// which let the compiler take the read-only path or move a load above the wait.  Tensor memory
// is allocated behind the wait and before the next may start: a CTA that holds it never waits for one that needs it.
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Whether a kernel that streams [rows][k] starts early.  On an SM where the previous kernel holds the shared memory it
// has next to no L1, which is what its loads in flight need; small ones gain all the same (577 x 768: norm, product,
// attention and quantisation in a row 27.5 -> 24.6 us; but norm and product of 4097 x 2048 62.1 -> 64.0).
inline bool mx_start_early(int rows, int k) { return (long long)rows * k <= 1 << 20; }

// Launches `kern` so (where `early`), in clusters of `cluster` CTAs along x.
template <typename... P, typename... A>
cudaError_t launch_early(bool early, void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t st, int cluster,
                         A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = early;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)cluster, 1u, 1u};
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P(args)...);
    if (e != cudaSuccess) cudaGetLastError();  // returned, not left for the next call to find
    return e;
}

// Thread i of them: 16 bytes of one of the last kt tiles, the scales of rows i % 32 + 0, 32, 64 and 96.
__device__ __forceinline__ void mx_pad_scales(uint8_t* scales, int rows, int kt, uint32_t i) {
    const uint32_t tile = i >> 5;
    if (tile >= (uint32_t)kt) return;
    const int n = (rows & 127) - (int)(i & 31);  // the operand has the four's rows where n > 0, 32, 64, 96
    uint8_t* p = scales + ((size_t)(rows >> 7) * kt + tile) * 512 + (i & 31) * 16;
    if (n <= 0) {
        *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
        for (int j = 1; j < 4; ++j)
            if (n <= 32 * j) reinterpret_cast<uint32_t*>(p)[j] = 0u;
    }
}

// Scale byte of a block from the largest of its values' absolute bits (as unsigned numbers, where
// infinity and NaN lie above every finite value).
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int e = (int)(amax_bits >> 23) - 2;
    return e > 0 ? (uint32_t)e : 0u;
}
// What the values are multiplied with: 2^(127 - e), exact for every finite block (e <= 252).
__device__ __forceinline__ float mx_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }
// 2^(e - 127): subnormal for 0, NaN for 255
__device__ __forceinline__ float mx_scale_value(uint32_t e) {
    return __uint_as_float(e == 0 ? 0x00400000u : (e == 255u ? 0x7fc00000u : e << 23));
}

// The two values of a byte of codes, as f16 pairs and in f32.
__device__ __forceinline__ uint32_t e2m1_halves(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 t;\n\t"
        "cvt.u8.u32 t, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, t;\n\t}\n"
        : "=r"(h)
        : "r"(byte));
    return h;
}
__device__ __forceinline__ float2 e2m1_values(uint32_t byte) {
    const uint32_t h = e2m1_halves(byte);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Codes of four or eight values of one block, column j in nibble j, rounded to the nearest (ties to the even
// code), saturating at 6; all zero where the block is not finite.
__device__ __forceinline__ uint32_t mx_codes4(const float (&v)[4], uint32_t e) {
    if (e == 255u) return 0u;
    const float inv = mx_inverse(e);
    uint32_t w;
    asm("{\n\t.reg .b8 t0, t1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
        "mov.b32 %0, {t0, t1, t0, t1};\n\t}\n"
        : "=r"(w)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv));
    return w & 0xffffu;
}
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], uint32_t e) {
    if (e == 255u) return 0u;
    const float2 inv = make_float2(mx_inverse(e), mx_inverse(e));
    const float2 a = __fmul2_rn(make_float2(v[0], v[1]), inv), b = __fmul2_rn(make_float2(v[2], v[3]), inv);
    const float2 c = __fmul2_rn(make_float2(v[4], v[5]), inv), d = __fmul2_rn(make_float2(v[6], v[7]), inv);
    uint32_t w;
    asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
        "mov.b32 %0, {t0, t1, t2, t3};\n\t}\n"
        : "=r"(w)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
    return w;
}

template <int N>
__device__ __forceinline__ uint32_t amax_bits(const float (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}

// ---- loads and stores of N = 4 or 8 neighbouring elements, 8 or 16 bytes at a time ----
template <typename T, int N>
struct VecN {
    static constexpr int WORDS = N * (int)sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (WORDS == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[0] = u.x; w[1] = u.y;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 u = reinterpret_cast<const uint4*>(p)[i / 4];
                w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    }
    // Two elements at a time, from an address on a boundary of two.
    __device__ __forceinline__ void load_pairs(const T* p) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + i);
                w[i] = u.x;
                w[i + 1] = u.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        }
    }
    // One at a time, the first `count` of them; zeros behind.
    __device__ __forceinline__ void load_some(const T* p, int count) {
        clear();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i >= count) continue;
            if constexpr (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
            else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
        }
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (__is_same(T, __half)) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    // the largest of the elements' absolute bits, as those of an f32
    __device__ __forceinline__ uint32_t amax() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
            // 16-bit magnitudes compare as unsigned numbers, two at a time
            uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
            for (int i = 1; i < WORDS; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            const uint32_t h = max(m & 0xffffu, m >> 16);
            if constexpr (__is_same(T, __half)) {
                if (h >= 0x7c00u) return 0x7f800000u;
                return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
            }
            return h << 16;
        }
    }
    __device__ __forceinline__ void set(const float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(v[i]);
            } else if constexpr (__is_same(T, __half)) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
    __device__ __forceinline__ void put(T* p) const {
        if constexpr (WORDS == 2) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4)
                reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
    }
    __device__ __forceinline__ void put_pairs(T* p) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(p + i) = make_uint2(w[i], w[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
        }
    }
    __device__ __forceinline__ void put_some(T* p, int count) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i >= count) continue;
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[i] = w[i];
            else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
    __device__ __forceinline__ static void store(T* p, const float (&v)[N]) {
        VecN x;
        x.set(v);
        x.put(p);
    }
};

// Elements that p lies behind a boundary of four of them.
template <typename T>
__device__ __forceinline__ int off_boundary(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) & 3);
}

// Two values rounded to T (16 bits), `a` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (__is_same(T, __half)) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (__is_same(T, __half)) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

#endif  // __CUDACC__

}  // namespace rfb
