// Product of two microscaled 4-bit operands, out = act(A B^T + bias) (formats in mx.cuh), on the
// block-scaled 4-bit path of the 5th-generation tensor cores: the codes and the scales are what
// tcgen05.mma.kind::mxf4 reads, nothing is unpacked.
//
//   warp 0      TMA producer (one lane): code tiles of 256 columns (128 bytes) and their scale tiles
//   warp 1      TMEM allocator; one lane copies the scales smem -> TMEM (tcgen05.cp) and issues
//               tcgen05.mma (M = 128 or, over a pair of SMs, 256; N = BN; K = 64), in that order:
//               the two are executed in issue order
//   warps 2..17 epilogue: accumulator -> registers -> bias, activation -> staging box -> TMA store
//               (four warps for each TMEM lane quadrant, a quarter of the columns each)
//
// Persistent CTAs, tiles round-robin, N fastest.  TMEM holds two accumulators so that the epilogue of
// one tile overlaps the products of the next.  With BN = 256 these and the scales do not fit 512
// columns, so the accumulators share 32 columns: accumulator 0 is columns [0, 256), accumulator 1
// [224, 480), the scales [480, 504).  The epilogue reads the shared 32 first, and the next tile starts
// once they are read.
//
// Scales in TMEM: the four bytes of a row (four blocks of 32 columns, two MMA steps) are one 32-bit
// cell, row r of 128 at lane r % 32, column r / 32, repeated in the four lane quadrants; the MMA step
// picks its pair of bytes by the id fields of the instruction descriptor.
#include "epilogue.cuh"
#include "mx.cuh"
#include "sm100.cuh"

#include <atomic>

namespace rfb {

namespace {

constexpr int BM = 128;
constexpr int BKE = 256;               // columns of a stage
constexpr int BKB = BKE / 2;           // its bytes in a row: one 128-byte swizzled row
constexpr int SF_GROUP = 1024;         // scale bytes of 128 rows x BKE columns
constexpr int BOX_BYTES = 2048;        // staging box of an epilogue warp: 32 rows x 64 bytes, or, where
constexpr int LOOSE_PITCH = 68;        // results do not leave by TMA, 32 rows this far apart

struct MxArgs {
    int M, N, K, ldo, act;
    const float* bias;
    void* out;
    int tma_out;       // the output leaves by TMA, or
    int row_boundary;  // bytes on whose boundaries all its rows lie: 8, 4 or 2
    int vec_out;  // its rows on boundaries of four elements
    int* err;     // the device's error word, set by a wait that runs out
};

template <int BN, bool CTA2>
struct MxCfg {
    static constexpr int TM = CTA2 ? 2 * BM : BM;
    static constexpr int B_ROWS = CTA2 ? BN / 2 : BN;  // rows of B this CTA loads
    static constexpr int BG = BN / 128;                // scale groups of B (a pair's CTAs need all of them)
    static constexpr int A_BYTES = BM * BKB;
    static constexpr int B_BYTES = B_ROWS * BKB;
    static constexpr int SF_BYTES = SF_GROUP * (1 + BG);
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
    static constexpr int NEPI = 16;
    static constexpr int THREADS = 64 + 32 * NEPI;
    static constexpr int OUT_STAGE = NEPI * 32 * LOOSE_PITCH;
    static constexpr int HC = BN / 4;                      // columns of an epilogue warp
    static constexpr int BIAS_BYTES = NEPI * HC * 4;       // bias of its columns
    static constexpr int TAIL = OUT_STAGE + BIAS_BYTES + 1024 + 256;
    static constexpr int STAGES = (232448 - TAIL) / STAGE_BYTES;
    static constexpr int SMEM = STAGES * STAGE_BYTES + TAIL;
    static constexpr bool SHARED = BN == 256;          // accumulators share columns
    static constexpr int ACC1 = SHARED ? 224 : BN;     // first column of accumulator 1
    static constexpr int T_SFA = ACC1 + BN;
    static constexpr int T_SFB = T_SFA + 8;
    static constexpr int TMEM_COLS = T_SFB + 8 * BG <= 512 && T_SFB + 8 * BG > 256 ? 512 : 256;
    static_assert(T_SFB + 8 * BG <= 512, "TMEM columns");
    static_assert(SMEM <= 232448, "shared memory");
};

// Instruction descriptor, kind::mxf4: A and B E2M1 (type 1 at bits 7 and 10), scales E8M0 (bit 23),
// N / 8 at bit 17, M / 128 at bit 27, the scales' byte ids at bits 29 (A) and 4 (B), K = 64.
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) |
           ((uint32_t)(M >> 7) << 27) | (sf_id << 29);
}

// Descriptor of a scale tile in shared memory for tcgen05.cp: 32 rows of 16 bytes, unswizzled, 8-row
// groups 128 bytes apart.
__device__ __forceinline__ uint64_t sf_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <bool CTA2>
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint64_t desc) {
    if constexpr (CTA2)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <bool CTA2>
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    if constexpr (CTA2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// NaN, which stands for a value that 4 bits cannot hold, passes every activation.
__device__ __forceinline__ void act_rows(float (&v)[32], int act) {
    if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const float2 w = gelu_erf2<true>(make_float2(v[j], v[j + 1]));
            v[j] = w.x;
            v[j + 1] = w.y;
        }
    } else if (act == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = positive<true>(v[j]);
    } else if (act == ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = act_fn<ACT_SILU>(v[j]);
    }
}

// 32 lanes x 16 columns of TMEM
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    __syncwarp();
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The staging box (rows of 64 bytes, LOOSE_PITCH apart) to rows m0.., columns n0.. of an output whose rows all lie on
// boundaries of a W (8, 4 or 2 bytes): one of them a lane.  (5273 x 12544 of K = 1274 by TMA 54 us, 12542 wide in words
// of 4 bytes 61, 12541 wide in words of 2 69; there 16-byte windows with single elements at the rows' ends took 79,
// pairs with single elements 82.)
template <typename T, typename W>
__device__ __forceinline__ void store_words(const uint8_t* box, const MxArgs& p, int m0, int n0, int lane) {
    constexpr int LANES = 64 / (int)sizeof(W), E = (int)sizeof(W) / (int)sizeof(T);  // lanes of a row, elements of a lane
    const int c = lane % LANES, n = n0 + c * E;
#pragma unroll 8
    for (int r = lane / LANES; r < 32; r += 32 / LANES) {
        if (m0 + r >= p.M) break;
        T* d = static_cast<T*>(p.out) + (size_t)(m0 + r) * p.ldo + n;
        const T* s = reinterpret_cast<const T*>(box + r * LOOSE_PITCH) + c * E;
        if (n + E <= p.N) {
            W x;
            if constexpr (sizeof(W) == 8) {
                x.x = reinterpret_cast<const uint32_t*>(s)[0];
                x.y = reinterpret_cast<const uint32_t*>(s)[1];
            } else {
                x = *reinterpret_cast<const W*>(s);
            }
            *reinterpret_cast<W*>(d) = x;
        } else {
#pragma unroll
            for (int i = 0; i + 1 < E; ++i)
                if (n + i < p.N) d[i] = s[i];
        }
    }
}

// 32 columns n0.. of this warp's 32 rows m0.. (one a lane) through its staging box: by TMA, which
// clips what lies behind the matrix, or, where it cannot, by the lanes.  A box row is 64 bytes: 32 columns of 16
// bits, or 16 of 32 in two turns.
// (16-byte stores of the lanes instead of TMA: 4096 x 8192 of K = 2048 46 us, GELU 55, against 38, 46.)
template <typename T>
__device__ __forceinline__ void store_chunk(const float (&v)[32], const CUtensorMap* map, uint8_t* box, uint32_t box_s,
                                            const MxArgs& p, int m0, int n0, int lane) {
    constexpr int COLS = 64 / (int)sizeof(T);
#pragma unroll
    for (int h = 0; h < 32 / COLS; ++h) {
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[h * 16 + j]);
            else w[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
        }
        const int n = n0 + h * COLS;
        if (p.tma_out) {
            if (elect_one()) bulk_wait_read<0>();  // the box's previous store has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
                st_shared_v4(swz64(box_s, lane, j), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            fence_async_smem();
            __syncwarp();
            if (elect_one()) {
                if (n < p.N && m0 < p.M)
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                                 "r"(box_s), "r"(n), "r"(m0)
                                 : "memory");
                bulk_commit();
            }
        } else {
            uint32_t* mine = reinterpret_cast<uint32_t*>(box + lane * LOOSE_PITCH);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) mine[j] = w[j];
            __syncwarp();
            if (n >= p.N) continue;
            if (p.row_boundary == 8) store_words<T, uint2>(box, p, m0, n, lane);
            else if (sizeof(T) == 4 || p.row_boundary == 4) store_words<T, uint32_t>(box, p, m0, n, lane);
            else if constexpr (sizeof(T) == 2) store_words<T, uint16_t>(box, p, m0, n, lane);
        }
    }
}

// CTA2: clusters of two CTAs.  Both producers' bytes count on rank 0's full[s]; rank 0 issues the
// pair's copies and products and commits to the empty[s] and tfull[a] of both; both epilogues
// arrive on rank 0's tempty.
template <int BN, bool CTA2, typename T>
__global__ void __launch_bounds__(MxCfg<BN, CTA2>::THREADS, 1)
k_mx_gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
          const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
          const __grid_constant__ CUtensorMap tmO, const MxArgs p) {
    using C = MxCfg<BN, CTA2>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + C::STAGES * C::A_BYTES;
    uint8_t* sSF = sB + C::STAGES * C::B_BYTES;
    uint8_t* out_stage = sSF + C::STAGES * C::SF_BYTES;
    float* bias_s = reinterpret_cast<float*>(out_stage + C::OUT_STAGE);
    uint64_t* full = reinterpret_cast<uint64_t*>(out_stage + C::OUT_STAGE + C::BIAS_BYTES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* tfull = empty + C::STAGES;
    uint64_t* tempty = tfull + 2;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
    volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CTA2 ? cluster_ctarank() : 0u;
    const int tile0 = CTA2 ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int tstep = CTA2 ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    const int n_tiles = (p.N + BN - 1) / BN;
    const int num_tiles = (p.M + C::TM - 1) / C::TM * n_tiles;
    const int num_kb = (p.K + BKE - 1) / BKE;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], (CTA2 ? 2 : 1) * 32 * C::NEPI);
        }
        *cta_abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        prefetch_tmap(&tmSA);
        prefetch_tmap(&tmSB);
    }
    wait_previous();
    if (warp == 1) {
        if constexpr (CTA2) tmem_alloc_pair(tmem_holder, C::TMEM_COLS);
        else tmem_alloc(tmem_holder, C::TMEM_COLS);
    }
    tc_fence_before();
    if constexpr (CTA2) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    let_next_start();

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = tile0; ok && tile < num_tiles; tile += tstep) {
                const int mt = tile / n_tiles, nt = tile - mt * n_tiles;
                const int arow = mt * C::TM + (int)rank * BM;
                const int brow = nt * BN + (int)rank * C::B_ROWS;
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait<CTA2>(&empty[stage], phase ^ 1, cta_abort, nullptr)) {
                        ok = false;
                        break;
                    }
                    uint8_t* a = sA + stage * C::A_BYTES;
                    uint8_t* b = sB + stage * C::B_BYTES;
                    uint8_t* sf = sSF + stage * C::SF_BYTES;
                    if constexpr (CTA2) {
                        if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE_BYTES);
                        const uint32_t fb = mapa_shared(smem_u32(&full[stage]), 0);
                        tma_load_2d_peer_bar(&tmA, fb, a, kb * BKB, arow);
                        tma_load_2d_peer_bar(&tmB, fb, b, kb * BKB, brow);
                        tma_load_2d_peer_bar(&tmSA, fb, sf, kb * (SF_GROUP / 4), arow >> 7);
                        tma_load_2d_peer_bar(&tmSB, fb, sf + SF_GROUP, kb * (SF_GROUP / 4), nt * C::BG);
                    } else {
                        mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
                        tma_load_2d(&tmA, &full[stage], a, kb * BKB, arow);
                        tma_load_2d(&tmB, &full[stage], b, kb * BKB, brow);
                        tma_load_2d(&tmSA, &full[stage], sf, kb * (SF_GROUP / 4), mt);
                        tma_load_2d(&tmSB, &full[stage], sf + SF_GROUP, kb * (SF_GROUP / 4), nt * C::BG);
                    }
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int stage = 0, local = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = tile0; ok && tile < num_tiles; tile += tstep, ++local) {
                const int acc = local & 1;
                // shared columns: the previous tile's are read; else: the tile before that is read
                if constexpr (C::SHARED)
                    ok = local == 0 || mbar_wait<CTA2>(&tempty[0], (local - 1) & 1, cta_abort, nullptr);
                else
                    ok = mbar_wait<CTA2>(&tempty[acc], ((local >> 1) & 1) ^ 1, cta_abort, nullptr);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + (acc ? C::ACC1 : 0);
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait<CTA2>(&full[stage], phase, cta_abort, nullptr)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(sA + stage * C::A_BYTES);
                    const uint32_t b0 = smem_u32(sB + stage * C::B_BYTES);
                    const uint32_t sf0 = smem_u32(sSF + stage * C::SF_BYTES);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // tiles of four blocks
                        sf_copy<CTA2>(tmem + C::T_SFA + 4 * i, sf_desc(sf0 + 512 * i));
#pragma unroll
                        for (int g = 0; g < C::BG; ++g)
                            sf_copy<CTA2>(tmem + C::T_SFB + 4 * (i * C::BG + g),
                                          sf_desc(sf0 + SF_GROUP * (1 + g) + 512 * i));
                    }
                    const int steps = min(BKE, p.K - kb * BKE);
#pragma unroll
                    for (int s = 0; s < BKE / 64; ++s) {
                        if (s * 64 >= steps) break;
                        umma_mxf4<CTA2>(d, sw128_kmajor_desc(a0 + s * 32), sw128_kmajor_desc(b0 + s * 32),
                                        idesc_mxf4(C::TM, BN, (s & 1) * 2), tmem + C::T_SFA + 4 * (s >> 1),
                                        tmem + C::T_SFB + 4 * C::BG * (s >> 1), (kb > 0 || s > 0) ? 1u : 0u);
                    }
                    if constexpr (CTA2) {
                        umma_commit_pair(smem_u32(&empty[stage]));
                        umma_commit_pair(mapa_shared(smem_u32(&empty[stage]), 1));
                    } else {
                        umma_commit(&empty[stage]);
                    }
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                if constexpr (CTA2) {
                    umma_commit_pair(smem_u32(&tfull[acc]));
                    umma_commit_pair(mapa_shared(smem_u32(&tfull[acc]), 1));
                } else {
                    umma_commit(&tfull[acc]);
                }
            }
        }
    } else {
        const int quad = warp & 3, part = (warp - 2) >> 2;
        constexpr int HC = C::HC, CH = HC / 32;  // columns and 32-column chunks of a warp
        uint8_t* box = out_stage + (warp - 2) * (p.tma_out ? BOX_BYTES : 32 * LOOSE_PITCH);
        const uint32_t box_s = smem_u32(box);
        float* my_bias = bias_s + (warp - 2) * HC;
        const uint32_t my_bias_s = smem_u32(my_bias);
        float next_bias[CH] = {};
        auto fetch_bias = [&](int tile) {
            const int n = (tile % n_tiles) * BN + part * HC + lane;
#pragma unroll
            for (int c = 0; c < CH; ++c) next_bias[c] = n + 32 * c < p.N ? p.bias[n + 32 * c] : 0.f;
        };
        if (p.bias && tile0 < num_tiles) fetch_bias(tile0);
        int local = 0;
        for (int tile = tile0; tile < num_tiles; tile += tstep, ++local) {
            const int mt = tile / n_tiles, nt = tile - mt * n_tiles;
            const int acc = local & 1;
            uint64_t* freed = &tempty[C::SHARED ? 0 : acc];
            auto release = [&]() {
                tc_fence_before();
                if constexpr (CTA2) mbar_arrive_cluster(mapa_shared(smem_u32(freed), 0));
                else mbar_arrive(freed);
            };
            if (p.bias) {
                __syncwarp();
#pragma unroll
                for (int c = 0; c < CH; ++c) my_bias[32 * c + lane] = next_bias[c];
                __syncwarp();
                if (tile + tstep < num_tiles) fetch_bias(tile + tstep);
            }
            if (!__all_sync(0xffffffffu, mbar_wait<CTA2>(&tfull[acc], (local >> 1) & 1, cta_abort, nullptr))) break;
            tc_fence_after();
            const int m0 = mt * C::TM + (int)rank * BM + quad * 32, nw = nt * BN + part * HC;
            const uint32_t tbase = tmem + ((uint32_t)(quad * 32) << 16) + (acc ? C::ACC1 : 0) + part * HC;
            // the shared columns are accumulator 0's last 32 and accumulator 1's first: the warps that
            // own them read them first
            const bool owns = part == (acc ? 0 : 3);
            const bool backwards = C::SHARED && acc == 0 && part == 3;
            if (C::SHARED && !owns) release();
            uint32_t raw[32];
            tmem_ld32(tbase + (backwards ? CH - 1 : 0) * 32, raw);
#pragma unroll 1
            for (int i = 0; i < CH; ++i) {
                const int ch = backwards ? CH - 1 - i : i;
                float v[32];
                tmem_wait_ld();
                if (C::SHARED ? (owns && i == 0) : i == CH - 1) release();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(raw[j]);
                // the next chunk is on its way while this one is worked on
                if (i + 1 < CH) tmem_ld32(tbase + (backwards ? ch - 1 : ch + 1) * 32, raw);
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 b = ld_shared_v4f(my_bias_s + (ch * 32 + j) * 4);
                        v[j] += b.x;
                        v[j + 1] += b.y;
                        v[j + 2] += b.z;
                        v[j + 3] += b.w;
                    }
                }
                act_rows(v, p.act);
                store_chunk<T>(v, &tmO, box, box_s, p, m0, nw + ch * 32, lane);
            }
        }
        if (p.tma_out && elect_one()) bulk_wait<0>();
    }
    linger_if_aborted(cta_abort);
    tc_fence_before();
    if constexpr (CTA2) cluster_sync();  // the peer may still arrive here, and the pair frees its TMEM together
    else __syncthreads();
    report_abort(cta_abort, p.err);
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CTA2) tmem_dealloc_pair(tmem, C::TMEM_COLS);
        else tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// ---- few rows of A, or few tiles ------------------------------------------------
//
// Few rows of A (tokens) leave a 128-row tile mostly empty, and what bounds the product is reading B
// (the weights) once; where there are few tiles, most SMs are idle.  So 128 rows of B are the M side of
// the tensor core, TN tokens its N side, and K is split over the CTAs of a cluster as far as the grid
// leaves SMs idle.  Each CTA multiplies its part of K and sends, to each other CTA of the cluster, the
// f32 sums of the tokens that are that one's to finish (one bulk copy between their shared memories);
// they are added in order of rank, so results do not change from run to run.
//   warp 0 TMA, warp 1 TMEM and tcgen05.mma, warps 2..9 epilogue
template <int TN>
struct FewCfg {
    static constexpr int A_BYTES = TN * BKB, B_BYTES = BM * BKB;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * SF_GROUP;
    // sums [token][row of B]: those of this CTA take the place of the stages, when they are done with;
    // those of the others [sender][token] have their own
    static constexpr int SUM_BYTES = BM * TN * 4;
    static constexpr int TAIL = SUM_BYTES + 1024 + 512;
    static constexpr int LEAST = (SUM_BYTES + STAGE_BYTES - 1) / STAGE_BYTES;  // stages that hold the sums
    static constexpr int MOST = (232448 - TAIL) / STAGE_BYTES;               // of a CTA alone on its SM
    static constexpr int HALF = ((233472 / 2 - 1024) - TAIL) / STAGE_BYTES;    // of two
    static constexpr int NEPI = 8;
    static constexpr int THREADS = 64 + 32 * NEPI;
    static constexpr int T_SFB = TN, T_SFA = TN + 8;  // TMEM columns behind the accumulator
    static constexpr int TMEM_COLS = TN + 16 <= 32 ? 32 : (TN + 16 <= 64 ? 64 : (TN + 16 <= 128 ? 128 : 256));
    static constexpr int smem(int stages) { return stages * STAGE_BYTES + TAIL; }
    static_assert(MOST >= LEAST && MOST >= 4 && (2 * MOST + 2) * 8 + 8 <= 512, "stages");
};

template <int TN, typename T>
__global__ void __launch_bounds__(FewCfg<TN>::THREADS)
k_mx_gemm_few(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const MxArgs p,
              const int parts, const int stages) {
    using C = FewCfg<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = smem;
    uint8_t* sA = sB + stages * C::B_BYTES;
    uint8_t* sSF = sA + stages * C::A_BYTES;
    float* sums = reinterpret_cast<float*>(sSF + stages * 2 * SF_GROUP);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sums) + C::SUM_BYTES);
    uint64_t* empty = full + C::MOST;
    uint64_t* done = empty + C::MOST;
    uint64_t* received = done + 1;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(received + 1);
    volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = parts > 1 ? (int)cluster_ctarank() : 0;
    const int tile = (int)blockIdx.x / parts;
    const int c0 = (int)blockIdx.y * TN;     // first token
    const int tokens = min(p.M - c0, TN);
    const int held = TN / parts;             // tokens [rank * held, rank * held + held) are this CTA's to finish
    const int mine = max(0, min(held, tokens - rank * held));
    const int num_kb = (p.K + BKE - 1) / BKE;
    const int kb0 = (int)((long long)num_kb * rank / parts), kb1 = (int)((long long)num_kb * (rank + 1) / parts);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        mbar_init(received, 1);
        mbar_arrive_expect_tx(received, (uint32_t)((parts - 1) * mine * BM * 4));
        *cta_abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        prefetch_tmap(&tmSA);
        prefetch_tmap(&tmSB);
    }
    wait_previous();
    if (warp == 1) tmem_alloc(tmem_holder, C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (parts > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // this CTA runs
    const uint32_t tmem = *tmem_holder;
    let_next_start();

    if (warp == 0) {
        if (elect_one()) {
            int s = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&empty[s], phase ^ 1, cta_abort, nullptr)) break;
                mbar_arrive_expect_tx(&full[s], C::STAGE_BYTES);
                tma_load_2d(&tmB, &full[s], sB + s * C::B_BYTES, kb * BKB, tile * BM);
                tma_load_2d(&tmSB, &full[s], sSF + s * 2 * SF_GROUP, kb * (SF_GROUP / 4), tile);
                tma_load_2d(&tmA, &full[s], sA + s * C::A_BYTES, kb * BKB, c0);
                tma_load_2d(&tmSA, &full[s], sSF + s * 2 * SF_GROUP + SF_GROUP, kb * (SF_GROUP / 4), c0 >> 7);
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            int s = 0;
            uint32_t phase = 0;
            bool all = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                all = mbar_wait(&full[s], phase, cta_abort, nullptr);
                if (!all) break;
                tc_fence_after();
                const uint32_t b0 = smem_u32(sB + s * C::B_BYTES), a0 = smem_u32(sA + s * C::A_BYTES);
                const uint32_t sf0 = smem_u32(sSF + s * 2 * SF_GROUP);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    sf_copy<false>(tmem + C::T_SFB + 4 * i, sf_desc(sf0 + 512 * i));
                    sf_copy<false>(tmem + C::T_SFA + 4 * i, sf_desc(sf0 + SF_GROUP + 512 * i));
                }
                const int steps = min(BKE, p.K - kb * BKE);
#pragma unroll
                for (int st = 0; st < BKE / 64; ++st) {
                    if (st * 64 >= steps) break;
                    umma_mxf4<false>(tmem, sw128_kmajor_desc(b0 + st * 32), sw128_kmajor_desc(a0 + st * 32),
                                     idesc_mxf4(BM, TN, (st & 1) * 2), tmem + C::T_SFB + 4 * (st >> 1),
                                     tmem + C::T_SFA + 4 * (st >> 1), (kb > kb0 || st > 0) ? 1u : 0u);
                }
                umma_commit(&empty[s]);
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (all) umma_commit(done);  // else nobody takes the sums for whole
        }
    }
    const int quad = warp & 3, row = quad * 32 + lane;
    float* own = reinterpret_cast<float*>(smem);  // over the stages
    bool ok = true;
    if (warp >= 2) {
        ok = __all_sync(0xffffffffu, mbar_wait(done, 0, cta_abort, nullptr));
        if (ok) {
            tc_fence_after();
#pragma unroll 1
            for (int c = (warp - 2) / 4 * 16; c < tokens; c += 32) {  // two warps for each TMEM lane quadrant
                float v[16];
                tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) own[(c + i) * BM + row] = v[i];
            }
        }
    }
    if (parts > 1) {
        fence_async_smem();
        __syncthreads();
        // every CTA of the cluster runs, and expects what it is sent
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (warp == 2 && ok && elect_one()) {
            for (int r = 0; r < parts; ++r) {
                const int count = max(0, min(held, tokens - r * held));
                if (r == rank || count == 0) continue;
                const uint32_t slot = smem_u32(sums + (rank * held) * BM);
                asm volatile(
                    "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                        mapa_shared(slot, r)),
                    "r"(smem_u32(own + r * held * BM)), "r"(count * BM * 4), "r"(mapa_shared(smem_u32(received), r))
                    : "memory");
            }
        }
        __syncwarp();
        if (warp >= 2 && ok) ok = __all_sync(0xffffffffu, mbar_wait<true>(received, 0, cta_abort, nullptr));
    }
    if (warp >= 2 && parts == 1) asm volatile("bar.sync 1, %0;" ::"n"(32 * C::NEPI) : "memory");  // every row's sums are written
    const int n = tile * BM + lane * 4;
    if (warp >= 2 && ok && n < p.N) {  // a warp finishes a token, a lane four of its columns
        float b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = p.bias && n + i < p.N ? p.bias[n + i] : 0.f;
        const uint32_t own_s = smem_u32(own + rank * held * BM + lane * 4), sums_s = smem_u32(sums + lane * 4);
        for (int c = warp - 2; c < mine; c += C::NEPI) {
            float x[4] = {};
            for (int r = 0; r < parts; ++r) {
                const float4 y = ld_shared_v4f(r == rank ? own_s + c * BM * 4 : sums_s + (r * held + c) * BM * 4);
                x[0] += y.x;
                x[1] += y.y;
                x[2] += y.z;
                x[3] += y.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] += b[i];
                if (p.act == ACT_GELU) x[i] = gelu_erf<true>(x[i]);
                else if (p.act == ACT_RELU) x[i] = positive<true>(x[i]);
                else if (p.act == ACT_SILU) x[i] = act_fn<ACT_SILU>(x[i]);
            }
            T* out = static_cast<T*>(p.out) + (size_t)(c0 + rank * held + c) * p.ldo + n;
            if (p.vec_out && n + 4 <= p.N) {
                VecN<T, 4>::store(out, x);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) out[i] = from_f32<T>(x[i]);
            }
        }
    }
    linger_if_aborted(cta_abort);
    __syncwarp();
    if (parts > 1) {
        cluster_sync();  // nobody still reads or writes another's shared memory,
        linger_if_aborted(cta_abort);  // but for what was sent to a CTA that no longer waits for it
    }
    tc_fence_before();
    __syncthreads();
    report_abort(cta_abort, p.err);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

bool make_map(CUtensorMap* m, CUtensorMapDataType type, const void* base, uint64_t cols, uint64_t rows, uint64_t pitch,
              uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_cols, box_rows}, estr[2] = {1, 1};
    return tensor_map_encode()(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// codes [rows][ceil(k / 32) * 16 bytes]
bool code_map(CUtensorMap* m, const uint8_t* codes, int rows, int k, int ld, int box_rows) {
    return make_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, ((uint64_t)k + 31) / 32 * 16, rows, ld, BKB, box_rows,
                    CU_TENSOR_MAP_SWIZZLE_128B);
}
// scale tiles as 32-bit words: [groups of 128 rows][tiles * 128 words]
bool scale_map(CUtensorMap* m, const uint8_t* scales, int rows, int k, int box_groups) {
    const uint64_t words = ((uint64_t)k + 127) / 128 * 128;
    return make_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, words, ((uint64_t)rows + 127) / 128, words * 4,
                    SF_GROUP / 4, box_groups, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct MxOperands {
    const uint8_t *a, *a_scales, *b, *b_scales;
    int lda, ldb;
};

template <typename T>
constexpr CUtensorMapDataType map_type() {
    return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : (__is_same(T, __half) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

// the dynamic shared memory limit of `kern`, set once for each device
template <typename K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t>& done, int dev) {
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load() & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

template <int BN, bool CTA2, typename T>
cudaError_t launch(const MxOperands& o, MxArgs p, int dev, int sms, cudaStream_t st) {
    using C = MxCfg<BN, CTA2>;
    static std::atomic<uint64_t> attr{0};
    cudaError_t e = allow_smem(k_mx_gemm<BN, CTA2, T>, C::SMEM, attr, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap ta, tb, tsa, tsb, to = {};
    if (!code_map(&ta, o.a, p.M, p.K, o.lda, BM) || !code_map(&tb, o.b, p.N, p.K, o.ldb, C::B_ROWS) ||
        !scale_map(&tsa, o.a_scales, p.M, p.K, 1) || !scale_map(&tsb, o.b_scales, p.N, p.K, C::BG))
        return cudaErrorInvalidValue;
    // a TMA store writes whole 16 bytes, also where the matrix ends inside them
    p.tma_out = ptr_aligned(p.out, 16) && (size_t)p.ldo * sizeof(T) % 16 == 0 && (size_t)p.N * sizeof(T) % 16 == 0 &&
                make_map(&to, map_type<T>(), p.out, p.N, p.M, (uint64_t)p.ldo * sizeof(T), 64 / sizeof(T), 32,
                         CU_TENSOR_MAP_SWIZZLE_64B);
    const uintptr_t low = (uintptr_t)p.out | (uintptr_t)((size_t)p.ldo * sizeof(T));
    p.row_boundary = low % 8 == 0 ? 8 : (low % 4 == 0 ? 4 : 2);
    const long long tiles = ((long long)p.M + C::TM - 1) / C::TM * (((long long)p.N + BN - 1) / BN);
    if (tiles > INT32_MAX - 1024) return cudaErrorInvalidValue;
    const int units = CTA2 ? sms / 2 : sms;
    const int grid = (int)(tiles < units ? tiles : units) * (CTA2 ? 2 : 1);
    return launch_early(true, k_mx_gemm<BN, CTA2, T>, dim3((unsigned)grid), C::THREADS, C::SMEM, st, CTA2 ? 2 : 1, ta, tb, tsa, tsb,
                        to, p);
}

// Parts of K: as many as there are SMs for, of two stages at least.  (Eight only within half of the SMs: a
// cluster needs them in one GPC, and sixteen such clusters wait for one another: 500 x 500 of K = 8192
// 17.6 us, in four parts 9.9.)
template <int TN>
int few_parts(const MxArgs& p, int sms) {
    const long long tiles = (((long long)p.N + BM - 1) / BM) * (((long long)p.M + TN - 1) / TN);
    const int num_kb = (p.K + BKE - 1) / BKE;
    int parts = 1;
    while (parts < 8 && tiles * parts * (parts < 4 ? 2 : 4) <= sms && num_kb >= 4 * parts) parts *= 2;
    return parts;
}
// Stages that the longest part has fewer than the whole K.
template <int TN>
int few_saved(const MxArgs& p, int sms) {
    const int num_kb = (p.K + BKE - 1) / BKE, parts = few_parts<TN>(p, sms);
    return num_kb - (num_kb + parts - 1) / parts;
}

template <int TN, typename T>
cudaError_t launch_few(const MxOperands& o, MxArgs p, int dev, int sms, cudaStream_t st) {
    using C = FewCfg<TN>;
    static std::atomic<uint64_t> attr{0};
    cudaError_t e = allow_smem(k_mx_gemm_few<TN, T>, C::smem(C::MOST), attr, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap ta, tb, tsa, tsb;
    if (!code_map(&ta, o.a, p.M, p.K, o.lda, TN) || !code_map(&tb, o.b, p.N, p.K, o.ldb, BM) ||
        !scale_map(&tsa, o.a_scales, p.M, p.K, 1) || !scale_map(&tsb, o.b_scales, p.N, p.K, 1))
        return cudaErrorInvalidValue;
    p.vec_out = ptr_aligned(p.out, 4 * sizeof(T)) && p.ldo % 4 == 0;
    const long long tiles = ((long long)p.N + BM - 1) / BM, row_tiles = ((long long)p.M + TN - 1) / TN;
    const int num_kb = (p.K + BKE - 1) / BKE, parts = few_parts<TN>(p, sms);
    // all of an SM's shared memory for stages where a CTA has it alone, half where two share it
    const int per = (num_kb + parts - 1) / parts, room = row_tiles * tiles * parts <= sms ? C::MOST : C::HALF;
    const int want = per < room ? per : room, stages = want > C::LEAST ? want : C::LEAST;
    if (tiles * parts > INT32_MAX) return cudaErrorInvalidValue;
    return launch_early(true, k_mx_gemm_few<TN, T>, dim3((unsigned)(tiles * parts), (unsigned)row_tiles), C::THREADS, C::smem(stages),
                        st, parts, ta, tb, tsa, tsb, p, parts, stages);
}

template <typename T>
cudaError_t dispatch(const MxOperands& o, MxArgs p, cudaStream_t st) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = op_error_word(dev, &p.err);
    if (e != cudaSuccess) return e;
    // A stage takes a CTA about 0.25 us; bringing the parts of TN tokens together 0.8 (32) to 4 us (128).  So K
    // is split where that saves TN / 8 stages or more: 1 x 4096 of K = 4096 5.3 us against 7.7, 32 x 4096 of
    // K = 4096 6.2 against 8.0, 64 x 256 of K = 16384 7.8 against 19.6, 300 x 300 of K = 16384 9.9 against 20.8;
    // left alone 64 x 64 of K = 1024 4.9 against 6.3, 500 x 1000 of K = 4096 8.5 against 9.7.  Up to 16 tokens gain
    // without a split, too (13 x 11008 of K = 4096 8.1 against 10.3).  (Each here without the early start.)
    if (p.M <= 16) return launch_few<16, T>(o, p, dev, sms, st);
    if (p.M <= 32 && few_saved<32>(p, sms) >= 4) return launch_few<32, T>(o, p, dev, sms, st);
    if (p.M <= 64 && few_saved<64>(p, sms) >= 8) return launch_few<64, T>(o, p, dev, sms, st);
    if (p.M > 64 && few_saved<128>(p, sms) >= 16) return launch_few<128, T>(o, p, dev, sms, st);
    // Narrow tiles until the wide ones cover the SMs (1616 x 1152 of K = 384: 4.7 us against 5.8).  Pairs
    // of SMs, where K is long and they need no more turns: a CTA then loads and reads half as much of B, which
    // is what bounds long K (18 TB/s from L2; 8192 x 8192 of K = 2048 70.9 us against 80.4, 4096 x 8192 35.7
    // against 38.3), but two epilogues wait for one another: of K = 1024 50.2 against 50.4, with GELU 61.8 against
    // 52.7; of K = 2048 with GELU the two are equal.
    const long long row_tiles = ((long long)p.M + 127) / 128, wide = row_tiles * (((long long)p.N + 255) / 256);
    if (wide < sms) return launch<128, false, T>(o, p, dev, sms, st);
    const long long pair_turns = ((row_tiles + 1) / 2 * (((long long)p.N + 255) / 256) + sms / 2 - 1) / (sms / 2);
    const int pair_k = p.act == ACT_GELU || p.act == ACT_SILU ? 4096 : 2048;
    if (p.K >= pair_k && pair_turns <= (wide + sms - 1) / sms) return launch<256, true, T>(o, p, dev, sms, st);
    return launch<256, false, T>(o, p, dev, sms, st);
}

}  // namespace

cudaError_t mx_gemm(const uint8_t* a, int lda, const uint8_t* a_scales, const uint8_t* b, int ldb,
                    const uint8_t* b_scales, int M, int N, int K, int act, const float* bias, void* out, int out_type,
                    int ldo, cudaStream_t st) {
    // K: the tensor core cuts the f32 sum, not rounds it, with every 64 columns: off by at most K 2^-29 of the sum of the
    // magnitudes, toward 0.  Up to this K that is half a step of bf16 (sums of one sign, scales far apart: 1.4e-5 at 2^16,
    // split over a cluster 3.3e-5 at 2^20).
    if (M < 0 || N < 0 || K < 1 || K > (1 << 21) || M > INT32_MAX - 255 || N > INT32_MAX - 255 || ldo < N ||
        !mx_type_ok(out_type) || act < ACT_NONE || act > ACT_SILU)
        return cudaErrorInvalidValue;
    if (M == 0 || N == 0) return cudaSuccess;
    if (!mx_codes_ok(a, lda, K) || !mx_codes_ok(b, ldb, K) || !a_scales || !b_scales || !ptr_aligned(a_scales, 16) ||
        !ptr_aligned(b_scales, 16) || !out || !ptr_aligned(out, mx_type_size(out_type)) || !ptr_aligned(bias, 4))
        return cudaErrorInvalidValue;
    if (!tensor_map_encode()) return cudaErrorNotSupported;
    const MxOperands o = {a, a_scales, b, b_scales, lda, ldb};
    const MxArgs p = {M, N, K, ldo, act, bias, out, 0, 0, 0, nullptr};
    switch (out_type) {
        case MX_F32: return dispatch<float>(o, p, st);
        case MX_F16: return dispatch<__half>(o, p, st);
        default: return dispatch<__nv_bfloat16>(o, p, st);
    }
}

}  // namespace rfb
