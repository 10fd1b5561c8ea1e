// The norms between one block of a transformer and the next, with the gate and the residual that
// stand between them:
//   x' = resid_scale x + gate * post(y)       h = pre(x')
// LayerNorm: (v - mean) / sqrt(mean (v - mean)^2 + eps) * w + b; RMSNorm: v / sqrt(mean v^2 + eps) * w.
// Everything between the loads and the stores is f32 in registers; h comes from x' before x' is
// rounded to the residual's type.  h leaves as a matrix, as a microscaled 4-bit operand (mx.cuh), or
// both.
//
// y and x are read once, x' and h written once, a dozen operations an element: bound by HBM.  A
// thread holds chunks of four columns (one 8- or 16-byte access of every operand, so a warp's accesses
// of either type are without gaps), C of them.  Rows of up to 512 columns belong to one warp each,
// longer ones to a CTA.  51712 x 384 f16 with an f32 residual: 37.5 us, 6.3 TB/s; 16 Mi elements of bf16 in and out:
// 25.7 us (5.2 TB/s) in rows of 1024, 27.0 of 2048, 26-28.5 of 4096, 31-32 of 8192, where the two sums' barriers
// show: one row's loads are in flight in a CTA.  Beyond, 1024 threads of 64 registers, some of which spill: 37 of
// 16384, 42 of 32768, 71 of 20000, which end inside the threads' chunks.
#include "mx.cuh"

namespace rfb {

namespace {

struct NormArgs {
    rfdetr_b200_block_norm p;
    int kt;             // scale tiles along k
    float inv_dim;
    uint32_t gate_magic;  // ceil(2^32 / gate_period) where row / gate_period is a multiplication with it, or 0
    unsigned pad_from;  // first CTA of those that write the scales' zeros
};

// Sum over the T threads of a row.  T > 32: through shared memory, `red` a buffer of this sum's own.
template <int T>
__device__ __forceinline__ float row_sum(float s, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if constexpr (T > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
        __syncthreads();
        // every warp adds the warps' sums in the same order
        s = red[threadIdx.x & (T / 32 - 1)];
#pragma unroll
        for (int o = T / 64; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    return s;
}

// First column of chunk c of thread t.
template <int T>
__device__ __forceinline__ int col_of(int c, int t) {
    return (c * T + t) * 4;
}

// Chunks of a row in their own type, 0 behind dim.  FULL: every column of the T * C chunks lies in the row
// and the row lies on a boundary of four; otherwise the accesses are as wide as the row's address allows.
// (The choice stands outside the loops, so that a row's loads are all on their way before the first is
// used: 16384 rows of 1023 bf16 60 us with it inside, 48 with it outside.)
template <typename S, int T, int C, bool FULL>
struct Row {
    VecN<S, 4> raw[C];
    // chunks c0 .. c0 + C - 1
    __device__ __forceinline__ void load(const S* row, int t, int dim, int c0 = 0) {
        const int off = FULL ? 0 : off_boundary(row);
        if (FULL || off == 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int n = col_of<T>(c0 + c, t);
                if (FULL || n + 4 <= dim) raw[c].load(row + n);
                else raw[c].clear();
            }
        } else if (off == 2) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int n = col_of<T>(c0 + c, t);
                if (n + 4 <= dim) raw[c].load_pairs(row + n);
                else raw[c].clear();
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) raw[c].load_some(row + col_of<T>(c0 + c, t), dim - col_of<T>(c0 + c, t));
        }
        if (!FULL && (dim & 3) != 0 && (off & 1) == 0) {  // the row's last one to three
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int n = col_of<T>(c0 + c, t);
                if (n < dim && n + 4 > dim) raw[c].load_some(row + n, dim - n);
            }
        }
    }
    __device__ __forceinline__ void get(int c, float (&v)[4]) const { raw[c].get(v); }
};

template <typename S, int T, int C, bool FULL>
__device__ __forceinline__ void store_row(S* row, const float (&v)[C][4], int t, int dim) {
    const int off = FULL ? 0 : off_boundary(row);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int n = col_of<T>(c, t);
        VecN<S, 4> x;
        x.set(v[c]);
        if (FULL || (off == 0 && n + 4 <= dim)) x.put(row + n);
        else if (off == 2 && n + 4 <= dim) x.put_pairs(row + n);
        else x.put_some(row + n, dim - n);
    }
}

// Columns behind dim to 0.
template <int T, bool FULL>
__device__ __forceinline__ void clear_behind(float (&v)[4], int c, int t, int dim) {
    if constexpr (!FULL) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col_of<T>(c, t) + j >= dim) v[j] = 0.f;
    }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 low(const float (&v)[4]) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ float2 high(const float (&v)[4]) { return make_float2(v[2], v[3]); }
__device__ __forceinline__ void put(float (&v)[4], float2 a, float2 b) { v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; }

// v = norm(v), LayerNorm or RMSNorm; columns behind dim stay 0.  Two values an instruction: a dozen
// operations an element would bound the 16-bit rows by the issue of instructions.
template <bool LAYER, int T, int C, bool FULL>
__device__ __forceinline__ void normalize(float (&v)[C][4], const float* w, const float* b, float eps, int dim,
                                          float inv_dim, int t, float* red) {
    constexpr bool kEarly = C <= 4;  // the weights' loads are issued before the sums where registers allow
    Row<float, T, kEarly ? C : 1, FULL> wr;
    Row<float, T, kEarly && LAYER ? C : 1, FULL> br;
    if constexpr (kEarly) {
        wr.load(w, t, dim);
        if constexpr (LAYER) br.load(b, t, dim);
    }
    if constexpr (LAYER) {
        float2 s = both(0.f);
#pragma unroll
        for (int c = 0; c < C; ++c) s = __fadd2_rn(s, __fadd2_rn(low(v[c]), high(v[c])));
        const float2 mean = both(-row_sum<T>(s.x + s.y, red) * inv_dim);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            put(v[c], __fadd2_rn(low(v[c]), mean), __fadd2_rn(high(v[c]), mean));
            clear_behind<T, FULL>(v[c], c, t, dim);  // no part of the variance
        }
    }
    float2 q = both(0.f);
#pragma unroll
    for (int c = 0; c < C; ++c) q = __ffma2_rn(high(v[c]), high(v[c]), __ffma2_rn(low(v[c]), low(v[c]), q));
    const float var = row_sum<T>(q.x + q.y, red + 32) * inv_dim + eps;
    float rstd = rsqrtf(var);
    rstd = fmaf(0.5f * rstd, fmaf(-var * rstd, rstd, 1.0f), rstd);  // one Newton step: to the last bit or so
    if (!(rstd > 0.f && rstd < 1e30f)) rstd = 1.0f / sqrtf(var);    // 0, infinity, NaN as they fall
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float wv[4], bv[4];
        if constexpr (kEarly) {
            wr.get(c, wv);
            if constexpr (LAYER) br.get(c, bv);
        } else {
            Row<float, T, 1, FULL> one;
            one.load(w, t, dim, c);
            one.get(0, wv);
            if constexpr (LAYER) {
                one.load(b, t, dim, c);
                one.get(0, bv);
            }
        }
        const float2 r = both(rstd);
        const float2 lo = __fmul2_rn(low(v[c]), r), hi = __fmul2_rn(high(v[c]), r);
        if constexpr (LAYER) put(v[c], __ffma2_rn(lo, low(wv), low(bv)), __ffma2_rn(hi, high(wv), high(bv)));
        else put(v[c], __fmul2_rn(lo, low(wv)), __fmul2_rn(hi, high(wv)));
    }
}

template <int T, int C, bool FULL>
__device__ __forceinline__ void normalize(float (&v)[C][4], int kind, const float* w, const float* b, float eps,
                                          int dim, float inv_dim, int t, float* red) {
    if (kind == NORM_LAYER) normalize<true, T, C, FULL>(v, w, b, eps, dim, inv_dim, t, red);
    else if (kind == NORM_RMS) normalize<false, T, C, FULL>(v, w, b, eps, dim, inv_dim, t, red);
}

// TY: type of y and h, TX: of the residual.
template <typename TY, typename TX, int T, int C, bool FULL>
__global__ void __launch_bounds__(T == 32 ? 128 : T)
k_block_norm(const NormArgs a) {
    constexpr int THREADS = T == 32 ? 128 : T;
    __shared__ float red[4 * 32];
    const rfdetr_b200_block_norm& p = a.p;
    let_next_start();
    wait_previous();
    if (blockIdx.x >= a.pad_from) {  // zeros of the scales behind the last row
        mx_pad_scales(static_cast<uint8_t*>(p.mx_scales), p.rows, a.kt, (blockIdx.x - a.pad_from) * THREADS + threadIdx.x);
        return;
    }
    const int t = threadIdx.x % T;
    const int row = (int)blockIdx.x * (THREADS / T) + (int)threadIdx.x / T;
    if (row >= p.rows) return;  // T = 32: a whole warp, and no barriers
    Row<TY, T, C, FULL> yr;
    // x is loaded with y, but where a CTA that wide has no registers for both: there, chunk by chunk
    constexpr bool kEarlyX = T * C <= 4096;
    Row<TX, T, kEarlyX ? C : 1, FULL> xr;
    const TX* x = static_cast<const TX*>(p.resid) + (size_t)row * p.ld_resid;
    yr.load(static_cast<const TY*>(p.y) + (size_t)row * p.ldy, t, p.dim);
    if constexpr (kEarlyX)
        if (p.resid) xr.load(x, t, p.dim);
    float y[C][4];
#pragma unroll
    for (int c = 0; c < C; ++c) yr.get(c, y[c]);
    normalize<T, C, FULL>(y, p.post, p.post_w, p.post_b, p.post_eps, p.dim, a.inv_dim, t, red);
    if (p.gate) {
        const int grow = !p.gate_period ? 0 : a.gate_magic ? (int)__umulhi((uint32_t)row, a.gate_magic) : row / p.gate_period;
        const float* g = p.gate + (size_t)grow * p.ld_gate;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            Row<float, T, 1, FULL> one;
            float gv[4];
            one.load(g, t, p.dim, c);
            one.get(0, gv);
            put(y[c], __fmul2_rn(low(y[c]), low(gv)), __fmul2_rn(high(y[c]), high(gv)));
        }
    }
    if (p.resid) {
        const float2 rs = both(p.resid_scale);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float xv[4];
            if constexpr (kEarlyX) {
                xr.get(c, xv);
            } else {
                xr.load(x, t, p.dim, c);
                xr.get(0, xv);
            }
            put(y[c], __ffma2_rn(rs, low(xv), low(y[c])), __ffma2_rn(rs, high(xv), high(y[c])));
        }
    }
    if (p.out_resid)
        store_row<TX, T, C, FULL>(static_cast<TX*>(p.out_resid) + (size_t)row * p.ld_out_resid, y, t, p.dim);
    normalize<T, C, FULL>(y, p.pre, p.pre_w, p.pre_b, p.pre_eps, p.dim, a.inv_dim, t, red + 64);
    if (p.out) store_row<TY, T, C, FULL>(static_cast<TY*>(p.out) + (size_t)row * p.ld_out, y, t, p.dim);
    if (!p.mx_codes) return;
    uint8_t* codes = static_cast<uint8_t*>(p.mx_codes) + (size_t)row * p.ld_mx;
    uint8_t* scales = static_cast<uint8_t*>(p.mx_scales);
    const int kpad = (p.dim + 31) & ~31;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        // eight lanes hold a block, a warp four
        const int n = col_of<T>(c, t);
        clear_behind<T, FULL>(y[c], c, t, p.dim);
        uint32_t m = amax_bits(y[c]);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
        const uint32_t e = mx_scale_of(m);
        uint32_t word = e << (8 * ((threadIdx.x >> 3) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        word |= __shfl_xor_sync(0xffffffffu, word, 16);
        if (FULL || n < kpad) *reinterpret_cast<uint16_t*>(codes + (n >> 1)) = (uint16_t)mx_codes4(y[c], e);
        if ((t & 31) == 0 && (n >> 7) < a.kt)
            *reinterpret_cast<uint32_t*>(scales + mx_scale_at(row, (n >> 7) * 4, a.kt)) = word;
    }
}

template <typename TY, typename TX, int T, int C>
cudaError_t launch(const rfdetr_b200_block_norm& p, bool aligned, cudaStream_t st) {
    constexpr int THREADS = T == 32 ? 128 : T;
    constexpr int ROWS = THREADS / T;
    NormArgs a;
    a.p = p;
    a.kt = (p.dim + 127) / 128;
    a.inv_dim = 1.0f / (float)p.dim;
    // exact while row * gate_period < 2^32
    a.gate_magic = p.gate_period > 1 && (uint64_t)p.rows * p.gate_period < 0x100000000ull
                       ? (uint32_t)((0x100000000ull + p.gate_period - 1) / p.gate_period) : 0u;
    a.pad_from = (unsigned)(((long long)p.rows + ROWS - 1) / ROWS);
    const long long pad = p.mx_codes && p.rows % 128 ? (mx_pad_threads(a.kt) + THREADS - 1) / THREADS : 0;
    if (a.pad_from + pad > INT32_MAX) return cudaErrorInvalidValue;
    auto kern = k_block_norm<TY, TX, T, C, false>;
    if (aligned && p.dim == T * C * 4) kern = k_block_norm<TY, TX, T, C, true>;
    return launch_early(mx_start_early(p.rows, p.dim), kern, dim3((unsigned)(a.pad_from + pad)), THREADS, 0, st, 1, a);
}

template <typename TY, typename TX>
cudaError_t dispatch(const rfdetr_b200_block_norm& p, bool aligned, cudaStream_t st) {
    const int d = p.dim;
    // Three to eight chunks a thread: fewer leave the two sums' barriers in the open (16 Mi elements of bf16 in
    // rows of 2048: 27.0 us with 128 threads, 32.1 with 256, 38.7 with 512), more the loads of one warp (27.7 with
    // 64, 49.6 with 32).  For one row it makes no difference: 4096 columns 2.9 us with 128 threads, 2.8 with 1024.
    if (d <= 128) return launch<TY, TX, 32, 1>(p, aligned, st);
    if (d <= 256) return launch<TY, TX, 32, 2>(p, aligned, st);
    if (d <= 384) return launch<TY, TX, 32, 3>(p, aligned, st);
    if (d <= 512) return launch<TY, TX, 32, 4>(p, aligned, st);
    if (d <= 768) return launch<TY, TX, 64, 3>(p, aligned, st);
    if (d <= 1024) return launch<TY, TX, 64, 4>(p, aligned, st);
    if (d <= 1280) return launch<TY, TX, 64, 5>(p, aligned, st);
    if (d <= 1536) return launch<TY, TX, 128, 3>(p, aligned, st);
    if (d <= 2048) return launch<TY, TX, 128, 4>(p, aligned, st);
    if (d <= 2560) return launch<TY, TX, 128, 5>(p, aligned, st);
    if (d <= 4096) return launch<TY, TX, 128, 8>(p, aligned, st);
    if (d <= 5120) return launch<TY, TX, 256, 5>(p, aligned, st);
    if (d <= 8192) return launch<TY, TX, 256, 8>(p, aligned, st);
    if (d <= 16384) return launch<TY, TX, 1024, 4>(p, aligned, st);
    return launch<TY, TX, 1024, 8>(p, aligned, st);
}

}  // namespace

cudaError_t block_norm(const rfdetr_b200_block_norm& p, cudaStream_t st) {
    auto norm_ok = [](int kind, const void* w, const void* b) {
        return kind == NORM_NONE || (kind == NORM_LAYER && w && b) || (kind == NORM_RMS && w);
    };
    if (!mx_type_ok(p.type) || p.rows < 0 || p.rows > INT32_MAX - 255 || p.dim < 1 || p.dim > 32768)
        return cudaErrorInvalidValue;
    if (p.rows == 0) return cudaSuccess;
    const bool has_x = p.resid || p.out_resid;
    if (has_x && p.resid_type != MX_F32 && p.resid_type != p.type) return cudaErrorInvalidValue;
    if (!p.y || p.ldy < p.dim || !norm_ok(p.post, p.post_w, p.post_b) || !norm_ok(p.pre, p.pre_w, p.pre_b))
        return cudaErrorInvalidValue;
    if (!(p.post_eps >= 0.f) || !(p.pre_eps >= 0.f)) return cudaErrorInvalidValue;
    if (p.gate && (p.gate_period < 0 || (p.gate_period > 0 && p.ld_gate < p.dim))) return cudaErrorInvalidValue;
    if ((p.resid && p.ld_resid < p.dim) || (p.out_resid && p.ld_out_resid < p.dim) || (p.out && p.ld_out < p.dim))
        return cudaErrorInvalidValue;
    if (!p.out_resid && !p.out && !p.mx_codes) return cudaErrorInvalidValue;
    if ((p.mx_codes != nullptr) != (p.mx_scales != nullptr)) return cudaErrorInvalidValue;
    if (p.mx_codes && (!mx_codes_ok(p.mx_codes, p.ld_mx, p.dim) || !ptr_aligned(p.mx_scales, 16)))
        return cudaErrorInvalidValue;
    const int sy = mx_type_size(p.type), sx = mx_type_size(p.resid_type);
    for (const void* f : {p.post_w, p.post_b, p.gate, p.pre_w, p.pre_b})
        if (!ptr_aligned(f, 4)) return cudaErrorInvalidValue;
    if (!ptr_aligned(p.y, sy) || !ptr_aligned(p.out, sy) || (has_x && (!ptr_aligned(p.resid, sx) || !ptr_aligned(p.out_resid, sx))))
        return cudaErrorInvalidValue;
    // whether every row of every operand lies on a boundary of four elements
    auto by4 = [](const void* q, long long ld, int size) { return !q || (ptr_aligned(q, 4 * size) && ld % 4 == 0); };
    const bool aligned = p.dim % 4 == 0 && by4(p.y, p.ldy, sy) && by4(p.resid, p.ld_resid, sx) &&
                     by4(p.out_resid, p.ld_out_resid, sx) && by4(p.out, p.ld_out, sy) && by4(p.post_w, 0, 4) &&
                     by4(p.post_b, 0, 4) && by4(p.gate, p.gate_period ? p.ld_gate : 0, 4) && by4(p.pre_w, 0, 4) &&
                     by4(p.pre_b, 0, 4);
    const bool wide = has_x && p.resid_type == MX_F32;
    switch (p.type) {
        case MX_F32: return dispatch<float, float>(p, aligned, st);
        case MX_F16: return wide ? dispatch<__half, float>(p, aligned, st) : dispatch<__half, __half>(p, aligned, st);
        default:
            return wide ? dispatch<__nv_bfloat16, float>(p, aligned, st) : dispatch<__nv_bfloat16, __nv_bfloat16>(p, aligned, st);
    }
}

}  // namespace rfb
