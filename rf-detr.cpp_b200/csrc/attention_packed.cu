// Attention over packed sequences of different lengths, causal or not, heads in groups that share
// their keys and values: for each sequence s (tokens cu[s] .. cu[s + 1]) and head h,
//   o = softmax(scale q k^T) v  over the keys of s (causal: up to the query's own position),
// with the running maximum and sum of the softmax over blocks of 128 keys.
//
// The rows of a tile are the `group` heads that share a key head, for TT = 128 / group tokens: row r
// is token r / group, head r % group of them, so short sequences and few tokens still fill the 128
// rows of the tensor core, and a key block serves every head that reads it.
//
// An item is two such tiles of one sequence and key head, the second over the TT tokens behind the
// first's; where tiles are few it is one, whose even key blocks are the first tile's below and whose odd
// ones the second's: each has its own maximum, sum and O, which the first joins at the end (in what
// follows "tile" is either); where sequences are one tile, it is just that.  The grid has a CTA for every
// item; a CTA that runs takes over the next one that has not started (cluster launch control), so that
// the loads and first products of an item run while the last one's results leave.
//   warps 0..3, 4..7  softmax of tile 0, 1: a thread owns a row, S from TMEM, exponentials in f32, P as
//                     packed 16-bit pairs back to TMEM; the reference maximum is raised, and O in TMEM
//                     rescaled, only when a row's maximum grows by more than 2^8, 2^4 in f16 (numerator
//                     and denominator share it)
//   warp 8            one lane issues tcgen05.mma: S_i = Q_i K^T and O_i += P_i V; while one tile's
//                     softmax runs, the other tile's products do, and P V starts on the first 64 keys of
//                     a block while the exponentials of the others are computed
//   warp 9            TMA: Q, K and V blocks into one ring
//   warp 10           finds the items' sequences, and hands them to the other warps
//   warp 11           overwrites with zeros the values behind a sequence's end, which belong to others (0
//                     times another sequence's infinity is not 0; keys are masked by position)
// TMEM, head_dim 128: S0 / P0 [0, 128), S1 / P1 [128, 256), O0, O1 behind them.  tcgen05.mma execute in
// issue order, so S_i of the next block, issued behind O_i += P_i V, overwrites P_i only when it was
// read, and its completion tells the softmax that O_i is at rest.
// head_dim 64: P has columns of its own, and S_i of the next block is issued as soon as this one's is
// read, before O_i += P_i V: tile by tile, so that the tiles run half a block apart (16 heads of 4096 tokens 103 us;
// both tiles' S first, which keeps them in step, 109).
#include "mx.cuh"
#include "sm100.cuh"
#include "softmax.cuh"

#include <atomic>
#include <cfloat>

namespace rfb {

namespace {

constexpr int TQ = 128;               // rows of a tile
constexpr int TK = 128;               // keys of a block
// The weights 2^(score - reference) enter the product with V as T, what the tensor core takes at its full rate (the error
// against 64 bits grows from 1.5e-3 to 2.0e-3 in bf16, from 2.1e-4 to 2.7e-4 in f16, relative 2-norms on random inputs,
// most of it the result's own rounding); the sums below them are those of the f32 weights (those of the rounded ones, which
// would cancel what all weights have in common, cost 4-10 %: prompts 52.6 -> 54.8 us, images 16.7 -> 18.1).  The
// reference is a row's maximum less LIFT, and moves when the maximum grows by more than RAISE (both log2).  bf16 rounds a
// weight by at most 2^-8 of it, however small.  f16 does so down to 2^-14 and holds less in steps of 2^-24: with the
// reference 2^11 below the maximum a weight is off by at most 2^-36 of its row's largest, and 2^19 of them, the most that a
// row has, together by 2^-17.  (Without it by 2^-25 each: 65535 weights of 2^-25.2, 1.7e-3 of the row, were 0.)
// The largest weight is 2^(LIFT + RAISE) = 2^15; f16 ends at 2^16.
template <typename T>
struct Weights {
    static constexpr bool HALF = __is_same(T, __half);
    static constexpr float LIFT = HALF ? 11.0f : 0.0f, RAISE = HALF ? 4.0f : 8.0f;
    // The reference of a maximum, and whether a row may keep its old one.  f16: rounded so that no weight is above
    // 2^15, however far the scores' f32 spacing is above 1.
    static __device__ __forceinline__ float reference(float top, float sl2) {
        return HALF ? __fadd_ru(__fmul_ru(top, sl2), -LIFT) : top * sl2;
    }
    static __device__ __forceinline__ bool keeps(float old, float cand) {
        return cand <= (HALF ? __fadd_rd(old, RAISE) : old + RAISE);
    }
};
// Registers a thread: 384 threads are launched with 168; 128 x 88 + 256 x 208 = 384 x 168.
constexpr int kLightRegs = 88, kSoftRegs = 208;

struct PackedArgs {
    void* o;
    const int32_t* cu;
    int n_seqs, tokens, ldo, kv_heads, group, tt, tiles, causal;
    int by_keys;  // the two softmax halves of a CTA share one tile's keys, not two tiles
    float sl2;  // scale / ln 2
    int* err;   // the device's error word, set by a wait that runs out
};

// What a CTA works on: rows [t0, t0 + tiles * tt) of the sequence whose tokens start at `start`.
struct Item {
    int start, len, t0, kvh;  // len 0: no more items
};

template <int HD>
struct PackedCfg {
    static constexpr int SUB = HD / 64;               // 64-column (128-byte) halves of a row
    static constexpr int TILE_BYTES = TK * HD * 2;    // of Q, K and V alike
    static constexpr int SLOTS = HD == 128 ? 5 : 8;   // K and V blocks in the ring
    static constexpr int TILES = (2 + SLOTS) * TILE_BYTES;
    static constexpr int SMEM = TILES + 1024 + 512 + TQ * 8;
    static constexpr int THREADS = 384;
    static constexpr bool APART = HD == 64;           // P beside S, not over it
    static constexpr int T_P = APART ? 2 * TK : 0;    // P_i at T_P + i * P_STEP
    static constexpr int P_STEP = APART ? TK / 2 : TK;
    static constexpr int T_O = APART ? 3 * TK : 2 * TK;
    // of 8 pairs of exponentials, those on the FMA pipe: where the products leave the MUFU the bound
    static constexpr int FMA_PAIRS = HD == 64 ? 2 : 0;
    static_assert(T_O + 2 * HD <= 512, "TMEM columns");
    static_assert(SMEM <= 232448, "shared memory");
};

// D f32, A and B f16 or bf16, B K-major or (b_mn) MN-major
template <typename T>
__host__ __device__ constexpr uint32_t idesc_16(int M, int N, bool b_mn) {
    const uint32_t fmt = __is_same(T, __half) ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

// V [keys][dims] as the MN-major operand: 64 dims wide swizzled rows, 8-key groups 1024 bytes apart, the
// second 64 dims one sub-tile (TK rows) further.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(TK * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The sequence that owns slot `slot`, with its first token and the next one's: slots of a sequence
// start at cu[s] / span + s, which leaves it at least ceil(length / span) of them, whatever the lengths.
// A warp looks at 32 sequences at a time.
__device__ __forceinline__ int sequence_of_slot(const int32_t* cu, int n_seqs, int span, int slot, int lane, int& first,
                                                int& next) {
    int lo = 0, hi = n_seqs;
    while (hi - lo > 31) {
        const int step = (hi - lo + 31) >> 5;
        const int s = lo + step * lane;
        const bool below = s < hi && cu[s] / span + s <= slot;
        const int n = __popc(__ballot_sync(0xffffffffu, below));
        lo += step * (n > 0 ? n - 1 : 0);
        hi = min(hi, lo + step);
    }
    const int s = lo + lane;
    const int c = s <= hi ? cu[s] : 0;
    const int n = __popc(__ballot_sync(0xffffffffu, s < hi && c / span + s <= slot));
    const int at = n > 0 ? n - 1 : 0;
    first = __shfl_sync(0xffffffffu, c, at);
    next = __shfl_sync(0xffffffffu, c, at + 1);
    return lo + at;
}

// Asks for a CTA of the grid that has not started; the answer (16 bytes) completes on `bar`.
__device__ __forceinline__ void ask_next_cta(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(answer)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// Its index along x, or -1 if there is none left.
__device__ __forceinline__ int next_cta(const void* answer) {
    int x, got;
    asm volatile(
        "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 a, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "selp.s32 %1, 1, 0, p;\n\t"
        "mov.s32 %0, -1;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, a;\n\t}\n"
        : "=r"(x), "=r"(got)
        : "r"(smem_u32(answer))
        : "memory");
    return got ? x : -1;
}

template <typename T, int HD>
__global__ void __launch_bounds__(PackedCfg<HD>::THREADS, 1)
k_attn_packed(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
              const __grid_constant__ CUtensorMap tmV, const PackedArgs p) {
    using C = PackedCfg<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;
    uint8_t* sKV = sQ + 2 * C::TILE_BYTES;
    uint8_t* answer = smem + C::TILES;                                    // 16 bytes
    Item* items = reinterpret_cast<Item*>(answer + 16);                    // [2]
    uint64_t* q_full = reinterpret_cast<uint64_t*>(items + 2);             // [2]
    uint64_t* q_free = q_full + 2;                                         // [2]
    uint64_t* kv_full = q_free + 2;                                        // [SLOTS]
    uint64_t* kv_empty = kv_full + C::SLOTS;                               // [SLOTS]
    uint64_t* s_full = kv_empty + C::SLOTS;                                // [2]
    uint64_t* s_free = s_full + 2;                                         // [2], P apart
    uint64_t* p_full = s_free + 2;                                         // [tile][half of the keys]
    uint64_t* pv_done = p_full + 4;                                        // [2]: an item's last, or (P apart) each
    uint64_t* o_free = pv_done + 2;                                        // [2]
    uint64_t* raw_full = o_free + 2;                                       // [SLOTS]: values that need zeros
    uint64_t* asked = raw_full + C::SLOTS;
    uint64_t* wanted = asked + 1;
    uint64_t* item_full = wanted + 1;                                      // [2]
    uint64_t* item_free = item_full + 2;                                   // [2]
    uint64_t* other_full = item_free + 2;                                  // by_keys: maximum and sum of tile 1
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(other_full + 1);
    volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_holder + 1);
    float2* other = reinterpret_cast<float2*>(answer + 512);               // [TQ]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 128);
            mbar_init(&p_full[2 * i], 128);
            mbar_init(&p_full[2 * i + 1], 128);
            mbar_init(&pv_done[i], 1);
            mbar_init(&o_free[i], 128);
            mbar_init(&item_full[i], 1);
            mbar_init(&item_free[i], 11);
        }
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
            mbar_init(&raw_full[i], 1);
        }
        mbar_init(other_full, 128);
        mbar_init(asked, 1);
        mbar_init(wanted, 1);
        *cta_abort = 0;
        fence_mbar_init();
    }
    wait_previous();
    if (warp == 8) tmem_alloc(tmem_holder, 512);
    // Item `index` of the grid; false if it is one of a sequence's slots that it does not need.
    const int span = p.tt * p.tiles;
    auto look_up = [&](int index, Item& it) {
        const int slot = index / p.kv_heads;
        int first, next;
        const int seq = sequence_of_slot(p.cu, p.n_seqs, span, slot, lane, first, next);
        it.kvh = index - slot * p.kv_heads;
        it.start = max(first, 0);
        it.len = min(next, p.tokens) - it.start;
        const int mine = slot - (first / span + seq), count = (it.len + span - 1) / span;
        it.t0 = (p.causal ? count - 1 - mine : mine) * span;  // longest rows first
        return it.len > 0 && mine >= 0 && mine < count;
    };
    Item own;
    bool found = false;
    if (warp == 10) found = look_up((int)blockIdx.x, own);  // while barriers and TMEM are set up
    if (warp == 9 && lane == 0) {
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    let_next_start();

    // The k-th item of this CTA for a warp of any role; false when there are no more.
    auto take = [&](int k, Item& it) -> bool {
        if (!__all_sync(0xffffffffu, mbar_wait(&item_full[k & 1], (k >> 1) & 1, cta_abort, nullptr))) return false;
        it = items[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_free[k & 1]);
        return it.len > 0;
    };
    // key blocks of an item, n[i] of them tile i's: causal, up to the last one that a row sees
    auto blocks_of = [&](const Item& it, int (&n)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int first = it.t0 + i * p.tt;
            n[i] = i >= p.tiles || first >= it.len ? 0 : ((p.causal ? min(it.len, first + p.tt) : it.len) + TK - 1) / TK;
        }
        const int all = max(n[0], n[1]);
        if (p.by_keys) {
            n[0] = (all + 1) >> 1;
            n[1] = all >> 1;
        }
        return all;
    };
    // the key block that is tile i's j-th
    auto block_at = [&](int i, int j) { return p.by_keys ? 2 * j + i : j; };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLightRegs));
        if (warp == 10) {
            int k = 0;
            bool ok = true;
            uint32_t phase = 0;
            while (true) {
                if (found) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&item_free[k & 1], ((k >> 1) & 1) ^ 1, cta_abort, nullptr));
                    if (!ok) break;
                    if (lane == 0) {
                        items[k & 1] = own;
                        mbar_arrive(&item_full[k & 1]);
                    }
                    // The next one is asked for when this one's last blocks are loaded: early enough to be
                    // there in time, late enough for other CTAs that are done sooner.
                    ok = __all_sync(0xffffffffu, mbar_wait(wanted, k & 1, cta_abort, nullptr));
                    if (!ok) break;
                    ++k;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(asked, 16);
                    ask_next_cta(answer, asked);
                }
                ok = __all_sync(0xffffffffu, mbar_wait(asked, phase, cta_abort, nullptr));
                if (!ok) break;
                phase ^= 1;
                const int index = next_cta(answer);
                if (index < 0) break;
                fence_async_smem();  // read before the next answer is written
                __syncwarp();
                found = look_up(index, own);
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&item_free[k & 1], ((k >> 1) & 1) ^ 1, cta_abort, nullptr));
            if (ok && lane == 0) {
                items[k & 1].len = 0;
                mbar_arrive(&item_full[k & 1]);
            }
        } else if (warp == 11) {
            Item it;
            int base = 0;         // blocks of the items before
            uint32_t phases = 0;  // of raw_full, a bit a slot
            for (int k = 0; take(k, it); ++k) {
                int nbi[2];
                const int nb = blocks_of(it, nbi), tail = it.len - (nb - 1) * TK;
                if (tail < TK) {
                    const int sl = (2 * (base + nb - 1) + 1) % C::SLOTS;
                    if (!__all_sync(0xffffffffu, mbar_wait(&raw_full[sl], (phases >> sl) & 1, cta_abort, nullptr))) break;
                    phases ^= 1u << sl;
                    const uint32_t dst = smem_u32(sKV + sl * C::TILE_BYTES);
                    const int chunks = (TK - tail) * 8;  // 16-byte chunks of the rows to clear, in one sub-tile
                    for (int c = 0; c < C::SUB; ++c)
                        for (int i = lane; i < chunks; i += 32)
                            st_shared_v4(dst + c * TK * 128 + tail * 128 + i * 16, 0, 0, 0, 0);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&kv_full[sl]);
                }
                base += nb;
            }
        } else if (warp == 9) {
            Item it;
            int idx = 0, used[2] = {0, 0};
            bool ok = true;
            for (int k = 0; ok && take(k, it); ++k) {
                int nbi[2];
                const int nb = blocks_of(it, nbi), tail = it.len - (nb - 1) * TK;
                if (elect_one()) {
                    for (int j = 0; ok && j < 2 * nb; ++j, ++idx) {
                        const int sl = idx % C::SLOTS;
                        uint8_t* dst = sKV + sl * C::TILE_BYTES;
                        ok = mbar_wait(&kv_empty[sl], ((idx / C::SLOTS) & 1) ^ 1, cta_abort, nullptr);
                        if (!ok) break;
                        // values that need zeros complete where warp 11 waits, which then fills kv_full
                        uint64_t* full = j == 2 * nb - 1 && tail < TK ? &raw_full[sl] : &kv_full[sl];
                        mbar_arrive_expect_tx(full, C::TILE_BYTES);
#pragma unroll
                        for (int c = 0; c < C::SUB; ++c)
                            tma_load_3d((j & 1) ? &tmV : &tmK, full, dst + c * TK * 128, c * 64, it.kvh,
                                        it.start + (j >> 1) * TK);
                        if (j == max(0, 2 * nb - 4)) mbar_arrive(wanted);
                        if (j > 0) continue;
                        for (int i = 0; i < 2; ++i) {  // behind the first keys: Q is free later than they are
                            if (nbi[i] == 0) continue;
                            if (used[i] > 0) ok = ok && mbar_wait(&q_free[i], (used[i] - 1) & 1, cta_abort, nullptr);
                            if (!ok) break;
                            ++used[i];
                            mbar_arrive_expect_tx(&q_full[i], p.tt * p.group * HD * 2);
#pragma unroll
                            for (int c = 0; c < C::SUB; ++c)
                                tma_load_4d(&tmQ, &q_full[i], sQ + i * C::TILE_BYTES + c * TQ * 128, c * 64, 0, it.kvh,
                                            it.start + it.t0 + (p.by_keys ? 0 : i * p.tt));
                        }
                    }
                }
                ok = __any_sync(0xffffffffu, !ok) == 0;
            }
        } else {
            constexpr uint32_t ID_S = idesc_16<T>(TQ, TK, false), ID_PV = idesc_16<T>(TQ, HD, true);
            Item it;
            int base = 0, sn[2] = {0, 0}, pn[2] = {0, 0}, used[2] = {0, 0};
            bool ok = true;
            for (int k = 0; ok && take(k, it); ++k) {
                int nbi[2];
                const int nb = blocks_of(it, nbi), steps = max(nbi[0], nbi[1]);
                if (elect_one()) {
                    auto slot_of = [&](int idx) { return (2 * base + idx) % C::SLOTS; };  // K_b 2b, V_b 2b + 1
                    auto wait_kv = [&](int idx) {
                        return mbar_wait(&kv_full[slot_of(idx)], ((2 * base + idx) / C::SLOTS) & 1, cta_abort, nullptr);
                    };
                    // tile i is the last (or only) user of its j-th block
                    auto last = [&](int i, int j) { return p.by_keys || i == 1 || nbi[1] <= j; };
                    auto issue_s = [&](int i, int j) {
                        const int slot = slot_of(2 * block_at(i, j));
                        if (!wait_kv(2 * block_at(i, j))) return false;
                        const uint32_t q = smem_u32(sQ + i * C::TILE_BYTES);
                        const uint32_t kk0 = smem_u32(sKV + slot * C::TILE_BYTES);
                        if (C::APART && sn[i] > 0 && !mbar_wait(&s_free[i], (sn[i] - 1) & 1, cta_abort, nullptr)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint32_t off = (kk >> 2) * TK * 128 + (kk & 3) * 32;
                            umma_f16(tmem + i * TK, sw128_kmajor_desc(q + off), sw128_kmajor_desc(kk0 + off), ID_S, kk > 0);
                        }
                        umma_commit(&s_full[i]);
                        if (j == nbi[i] - 1) umma_commit(&q_free[i]);
                        if (last(i, j)) umma_commit(&kv_empty[slot]);
                        ++sn[i];
                        return true;
                    };
                    auto issue_pv = [&](int i, int j, int h) {  // keys [64 h, 64 h + 64) of the block
                        const uint32_t v = smem_u32(sKV + slot_of(2 * block_at(i, j) + 1) * C::TILE_BYTES);
                        tc_fence_after();
#pragma unroll
                        for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                            umma_f16_ts(tmem + C::T_O + i * HD, tmem + C::T_P + i * C::P_STEP + kk * 8,
                                        v_desc(v + kk * 2048), ID_PV, (j > 0 || kk > 0) ? 1u : 0u);
                    };
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!ok || nbi[i] == 0) continue;
                        ok = mbar_wait(&q_full[i], used[i] & 1, cta_abort, nullptr) && issue_s(i, 0);
                    }
                    for (int j = 0; ok && j < steps; ++j) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (!ok || j >= nbi[i]) continue;
                            if (j == 0 && used[i] > 0) ok = mbar_wait(&o_free[i], (used[i] - 1) & 1, cta_abort, nullptr);
                            if constexpr (C::APART)
                                if (ok && j + 1 < nbi[i]) ok = issue_s(i, j + 1);
                            if (ok) ok = wait_kv(2 * block_at(i, j) + 1);
                            if (ok) ok = mbar_wait(&p_full[2 * i], pn[i] & 1, cta_abort, nullptr);
                            if (!ok) continue;
                            issue_pv(i, j, 0);
                            ok = mbar_wait(&p_full[2 * i + 1], pn[i] & 1, cta_abort, nullptr);
                            if (!ok) continue;
                            issue_pv(i, j, 1);
                            ++pn[i];
                            if (last(i, j)) umma_commit(&kv_empty[slot_of(2 * block_at(i, j) + 1)]);
                            if (C::APART || j + 1 == nbi[i]) umma_commit(&pv_done[i]);
                            else ok = issue_s(i, j + 1);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) used[i] += nbi[i] > 0;
                    base += nb;
                }
                ok = __any_sync(0xffffffffu, !ok) == 0;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int tile = warp >> 2, quad = warp & 3;
        const int row = quad * 32 + lane;
        const int row_tok = row / p.group, row_head = row - row_tok * p.group;
        const uint32_t lanebase = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + tile * TK + lanebase, tP = tmem + C::T_P + tile * C::P_STEP + lanebase,
                       tO = tmem + C::T_O + tile * HD + lanebase;
        const float sl2 = p.sl2;
        Item it;
        int sn = 0, done = 0, merged = 0;  // S blocks, pv_done and other_full phases so far
        bool ok = true;
        for (int k = 0; ok && take(k, it); ++k) {
            int nbi[2];
            blocks_of(it, nbi);
            const int my_nb = nbi[tile];
            if (my_nb == 0) continue;
            const int tok = it.t0 + (p.by_keys ? 0 : tile * p.tt) + row_tok;  // position in the sequence
            const bool valid = row_tok < p.tt && tok < it.len;
            const int limit = p.causal && valid ? tok + 1 : it.len;  // keys this row sees
            // Finite at first, so that keys whose scores are all -infinity leave it, l and O as they are.
            float m = -FLT_MAX, l = 0.f;
            for (int j = 0; j < my_nb; ++j, ++sn) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[tile], sn & 1, cta_abort, nullptr));
                if (!ok) break;
                tc_fence_after();
                uint32_t r[4][32];
#pragma unroll
                for (int h = 0; h < 4; ++h) tmem_ld32(tS + 32 * h, r[h]);
                tmem_wait_ld();
                if constexpr (C::APART) {
                    tc_fence_before();
                    mbar_arrive(&s_free[tile]);
                }
                const int seen = limit - block_at(tile, j) * TK;  // of this block's keys
                if (__any_sync(0xffffffffu, seen < TK)) {
#pragma unroll
                    for (int h = 0; h < 4; ++h)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (32 * h + e >= seen) r[h][e] = __float_as_uint(-INFINITY);
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int h = 0; h < 4; h += 2)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        mx4[e & 3] = fmax3_nan(mx4[e & 3], __uint_as_float(r[h][e]), __uint_as_float(r[h + 1][e]));
                const float m_cand =
                    Weights<T>::reference(fmax3_nan(fmax3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], -INFINITY), sl2);
                const float m_new = Weights<T>::keeps(m, m_cand) ? m : m_cand;  // the first finite one is always taken, and NaN
                const float alpha = ex2(m - m_new);
                if constexpr (C::APART) {
                    if (j > 0) {  // the previous product has read P, and O is at rest
                        ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[tile], done & 1, cta_abort, nullptr));
                        if (!ok) break;
                        ++done;
                        tc_fence_after();
                    }
                }
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f && valid)) {
                    uint32_t o[32];
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        tmem_ld32(tO + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 y = __fmul2_rn(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])),
                                                        make_float2(alpha, alpha));
                            o[e] = __float_as_uint(y.x);
                            o[e + 1] = __float_as_uint(y.y);
                        }
                        tmem_st32(tO + c, o);
                    }
                }
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 sl2v = make_float2(sl2, sl2), negm = make_float2(-m_new, -m_new);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t pk[32];  // column c of P holds keys 2c, 2c + 1
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 a = __ffma2_rn(
                                make_float2(__uint_as_float(r[2 * g + h][e]), __uint_as_float(r[2 * g + h][e + 1])), sl2v,
                                negm);
                            const bool on_fma = ((e >> 1) & 7) >= 8 - C::FMA_PAIRS;
                            const float2 x = on_fma ? exp2_fma2<true>(a) : make_float2(ex2(a.x), ex2(a.y));
                            sum[h] = __fadd2_rn(sum[h], x);
                            pk[h * 16 + (e >> 1)] = pack2<T>(x.x, x.y);
                        }
                    }
                    tmem_st32(tP + 32 * g, pk);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&p_full[2 * tile + g]);
                }
                l = l * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                m = m_new;
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[tile], done & 1, cta_abort, nullptr));
            if (!ok) break;
            ++done;
            tc_fence_after();
            // by_keys: tile 1 hands its maximum and sum over, tile 0 adds its O to its own; o = own O + share O_1
            const bool both = p.by_keys && nbi[1] > 0;
            float own = 1.0f / l, share = 0.f;
            if (both) {
                if (tile == 1) {
                    other[row] = make_float2(m, l);
                    tc_fence_before();
                    mbar_arrive(other_full);
                    continue;
                }
                ok = __all_sync(0xffffffffu, mbar_wait(other_full, merged & 1, cta_abort, nullptr));
                if (!ok) break;
                ++merged;
                tc_fence_after();
                const float2 ml = other[row];
                const float top = fmaxf(m, ml.x);
                own = ex2(m - top);
                share = ex2(ml.x - top);
                const float inv = 1.0f / (l * own + ml.y * share);
                own *= inv;
                share *= inv;
            }
            T* out = static_cast<T*>(p.o) + (size_t)(it.start + tok) * p.ldo + (size_t)(it.kvh * p.group + row_head) * HD;
#pragma unroll
            for (int c = 0; c < HD; c += 64) {
                uint32_t o[2][32];
                tmem_ld32(tO + c, o[0]);
                tmem_ld32(tO + c + 32, o[1]);
                tmem_wait_ld();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[h][e] = __float_as_uint(__uint_as_float(o[h][e]) * own);
                    if (both) {
                        uint32_t y[32];
                        tmem_ld32(tO + HD + c + 32 * h, y);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            o[h][e] = __float_as_uint(fmaf(__uint_as_float(y[e]), share, __uint_as_float(o[h][e])));
                    }
                }
                if (c + 64 == HD) {
                    tc_fence_before();
                    mbar_arrive(&o_free[tile]);
                    if (both) mbar_arrive(&o_free[1]);
                }
                if (!valid) continue;
#pragma unroll
                for (int e = 0; e < 64; e += 8) {
                    const uint32_t* x = &o[e >> 5][e & 31];
                    uint4 u;
                    u.x = pack2<T>(__uint_as_float(x[0]), __uint_as_float(x[1]));
                    u.y = pack2<T>(__uint_as_float(x[2]), __uint_as_float(x[3]));
                    u.z = pack2<T>(__uint_as_float(x[4]), __uint_as_float(x[5]));
                    u.w = pack2<T>(__uint_as_float(x[6]), __uint_as_float(x[7]));
                    *reinterpret_cast<uint4*>(out + c + e) = u;
                }
            }
        }
    }
    linger_if_aborted(cta_abort);
    tc_fence_before();
    __syncthreads();
    report_abort(cta_abort, p.err);
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T>
bool make_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
              const cuuint32_t* box) {
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return tensor_map_encode()(m, __is_same(T, __half) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                    (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
cudaError_t launch(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv, PackedArgs p, int max_len,
                   cudaStream_t st) {
    using C = PackedCfg<HD>;
    static std::atomic<uint64_t> attr{0};
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = op_error_word(dev, &p.err);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr.load() & bit)) {
        e = cudaFuncSetAttribute(k_attn_packed<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        attr.fetch_or(bit);
    }
    p.tt = TQ / p.group;
    // Two tiles of a CTA read each block once.  One, whose keys go to the two halves in turn, has half the chain, and
    // its sums are joined at the end: where two would leave half of the SMs idle (6 heads of 1601 tokens, head_dim 64:
    // 17.8 us against 21.9 with a half idle, 2 of 6000, causal: 47 against 76), and causal, where the pairs are of
    // all lengths, while they start all at once (8 heads of 3000 tokens 28 against 48; 16 of 4096, twice as many
    // as SMs, 69 against 64; not causal, 16 heads of 1601 28 against 26).  One block is left whole.
    const long long pairs = ((long long)p.tokens / (2 * p.tt) + 1) * p.kv_heads;
    p.tiles = max_len <= p.tt || (p.causal ? 1 : 2) * pairs <= sms ? 1 : 2;
    p.by_keys = p.tiles == 1 && max_len > TK;
    const long long slots = (long long)p.tokens / (p.tt * p.tiles) + p.n_seqs;
    if (slots * p.kv_heads > INT32_MAX) return cudaErrorInvalidValue;
    const cuuint64_t qd[4] = {HD, (cuuint64_t)p.group, (cuuint64_t)p.kv_heads, (cuuint64_t)p.tokens};
    const cuuint64_t qs[3] = {HD * 2, (cuuint64_t)p.group * HD * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t qb[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)p.tt};
    const cuuint64_t kd[3] = {HD, (cuuint64_t)p.kv_heads, (cuuint64_t)p.tokens};
    const cuuint64_t ks[2] = {HD * 2, (cuuint64_t)ldk * 2}, vs[2] = {HD * 2, (cuuint64_t)ldv * 2};
    const cuuint32_t kb[3] = {64, 1, TK};
    CUtensorMap mq, mk, mv;
    if (!make_map<T>(&mq, q, 4, qd, qs, qb) || !make_map<T>(&mk, k, 3, kd, ks, kb) || !make_map<T>(&mv, v, 3, kd, vs, kb))
        return cudaErrorInvalidValue;
    return launch_early(true, k_attn_packed<T, HD>, dim3((unsigned)(slots * p.kv_heads)), C::THREADS, C::SMEM, st, 1, mq, mk, mv, p);
}

}  // namespace

cudaError_t attention_packed(const void* q, const void* k, const void* v, int ldq, int ldk, int ldv, void* o, int ldo,
                             int type, const int32_t* cu_seqlens, int n_seqs, int tokens, int max_len, int heads,
                             int kv_heads, int head_dim, int causal, float scale, cudaStream_t st) {
    // max_len: the tensor core cuts the f32 sums of P V, not rounds them, with every 16 keys: off by at most max_len 2^-27 of
    // the weighted mean of |v|, toward 0.  Up to this length that is half a step of bf16 (equal weights, values of one sign:
    // 1.7e-4 at 2^16, 1.4e-3 at 2^18, 6.5e-3 at 2^20; O in two parts would need the TMEM that the scores have).
    if ((type != MX_F16 && type != MX_BF16) || (head_dim != 64 && head_dim != 128) || n_seqs < 0 || tokens < 0 ||
        max_len < 0 || max_len > (1 << 19) || heads < 1 || kv_heads < 1 || heads % kv_heads || heads / kv_heads > 128 ||
        heads > INT32_MAX / 128 || !(scale > 0.f) || scale > 2e38f)  // scale / ln 2 is finite
        return cudaErrorInvalidValue;
    if (ldq < heads * head_dim || ldo < heads * head_dim || ldk < kv_heads * head_dim || ldv < kv_heads * head_dim ||
        ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8)
        return cudaErrorInvalidValue;
    if (n_seqs == 0 || tokens == 0 || max_len == 0) return cudaSuccess;
    for (const void* x : {q, k, v, (const void*)o})
        if (!x || !ptr_aligned(x, 16)) return cudaErrorInvalidValue;
    if (!cu_seqlens || !ptr_aligned(cu_seqlens, 4)) return cudaErrorInvalidValue;
    if (!tensor_map_encode()) return cudaErrorNotSupported;
    const PackedArgs p = {o, cu_seqlens, n_seqs, tokens, ldo, kv_heads, heads / kv_heads, 0, 0, causal != 0, 0,
                          scale * 1.4426950408889634f, nullptr};
    if (type == MX_F16)
        return head_dim == 64 ? launch<__half, 64>(q, k, v, ldq, ldk, ldv, p, max_len, st)
                              : launch<__half, 128>(q, k, v, ldq, ldk, ldv, p, max_len, st);
    return head_dim == 64 ? launch<__nv_bfloat16, 64>(q, k, v, ldq, ldk, ldv, p, max_len, st)
                          : launch<__nv_bfloat16, 128>(q, k, v, ldq, ldk, ldv, p, max_len, st);
}

}  // namespace rfb
