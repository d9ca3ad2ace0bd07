// Softmax cross entropy of a linear output layer, logits never kept, and its gradients.
//
//   logits = H W^T          H: T x D tokens, W: V x D, both bf16; fp32 products in TMEM
//   loss_t = lse_t - logits(t, target_t),   lse_t = log sum_v exp logits(t, v)
//   G(t, v) = g_t (exp(logits(t, v) - lse_t) - [v = target_t])
//   dH = G W,   dW = G^T H
//
// GEMM -> row softmax -> GEMM once more (attention.cu), with a second product on the way back: the
// forward pass keeps a running maximum and sum per row in the epilogue of the product, the backward
// pass forms the product again, turns it into G in the epilogue and feeds G to two more products.
//
// Bound: tensor pipe, 2 T V D operations forward and 6 T V D backward (the product again, dH, dW);
// with few tokens the reading of W.  All four products run in one kernel template on CTA pairs (256 x
// 256 tiles, tcgen05.mma cta_group::2, TMA ring, two accumulators in TMEM; the structure of
// gemm_bf16_2cta.cu), which differs from that one in its epilogues and in operands that are read with
// the MN dimension contiguous: W as the K x N operand of dH, G as the M x K operand and H as the
// K x N operand of dW.  No operand is ever transposed in memory.
//
// Only tokens that count take part: a first kernel lists them, a second one packs their rows of H
// (T x D x 4 bytes of traffic, 0.1 % of the products' time at 8192 x 131072 x 4096).  Ignored tokens
// then cost nothing, and what their rows hold (NaN, infinities) reaches no gradient; a product with
// zeros in G would spread it.  The number of counted tokens stays on the device: kernels read it and
// take that many rows of tiles.
//
// G goes through memory in pieces of the vocabulary (kPieceBytes), as bf16.  That rounding is half a
// step, 2^-9 relative at most, independent from entry to entry; the factor that all tokens share (the
// largest |g_t|) is kept out of it and applied to the fp32 sums, since a common factor's rounding
// would not average out: the entry at the target, near -g_t, would be off by the same share everywhere.
#include <algorithm>
#include <math.h>

#include "common.cuh"
#include "smem_plan.hpp"

namespace gb200 {
namespace {

constexpr int BN = 256, BK = 64, HALF = 128;
constexpr int CHUNK_BYTES = 64 * BK * 2;    // MN-major operand: 64 columns x 64 K rows, 128 bytes per row
constexpr int GROUP_M = 8;                  // tile rows per rasterisation group
constexpr int EPI_WARPS = 8;                // two per quarter of the TMEM lanes, 128 columns each
constexpr int NUM_THREADS = 64 + 32 * EPI_WARPS;
constexpr int STORE_BYTES = 128 * 64 * 2;   // staging tile of a TMA store: 128 rows x 64 columns
constexpr int SEGMENT = 16;                 // K blocks that kLse adds up in the tensor cores at a time

enum Mode { kLse, kProb, kDh, kDw };

// PAIR: 256 x 256 tiles on two CTAs, each of which stages its half of A and of B.  Otherwise 128 x 256
// tiles on one CTA: with at most 128 tokens the pair would spend half its MMA time on rows that do not
// exist, and with few tokens that time, not the reading of W, was the longer (65536 x 4096, one
// token: tensor pipe 74 % active at 58 % of the DRAM rate, 126 us).
template <int MODE, bool PAIR>
struct Shape {
    static constexpr bool STORE = MODE == kProb || MODE == kDw;    // results leave through shared memory
    static constexpr int BM = PAIR ? 256 : 128;
    static constexpr int A_BYTES = HALF * BK * 2, B_BYTES = (PAIR ? HALF : BN) * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = PAIR ? (STORE ? 5 : 6) : (STORE ? 3 : 4);
    static constexpr smem::XentLayout layout = smem::xent_layout(STAGES, STAGE_BYTES, STORE ? 4 * STORE_BYTES : 0);
};

// G of one piece of the vocabulary: large enough that a piece fills the SMs many times over, small
// beside W and dW (1 GiB each at 131072 x 4096).
constexpr int64_t kPieceBytes = 256ll << 20;
constexpr int64_t kSlabBytes = 512ll << 20;   // most that split sums of dH may take

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;

// What the first kernel leaves for the others.
struct Scalars {
    int count;        // tokens that count
    int bad;          // tokens whose target is neither in [0, V) nor ignore_index
    float factor;     // common factor of the gradients
    float largest;    // largest |g_t|
};

struct Args {
    const Scalars *sc;
    int m, n, k;               // extents; the one that is the number of counted tokens is read from sc
    int b_row0;                // row of the B operand's tensor map where this piece starts
    int v0;                    // first vocabulary row of this piece
    const int *target;         // [count]
    // kLse
    float2 *partial;           // [2 per tile column][ld_partial]: maximum (times log2 e) and sum
    int64_t ld_partial;
    int part0;                 // first slot of this piece
    int running;               // one row of tiles: a unit keeps its maximum and sum over all its tiles
    float *target_logit;       // [count]
    // kProb
    const float *lse;          // [count]
    const float *weight;       // [count], NULL: all equal
    // kDh
    float *slab;               // [splits][rows_pad][n], fp32 sums over the pieces so far
    int64_t slab_stride, ld_slab;
    int splits;
    int first, last;           // first piece: the slab holds nothing yet; last: dH is written (splits == 1)
    const int *rows;           // [count]: token of a packed row
    // results: G, dH, or this piece's rows of dW
    __nv_bfloat16 *out;
    int64_t ldo;
    int tma_out;               // kProb, kDw: through tmap_out (addresses and pitch allow it)
    int *status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 32 consecutive bf16 of a row; `n` of them are inside the matrix.
__device__ __forceinline__ void store_row32(__nv_bfloat16 *dst, const float (&v)[32], int n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(dst);
    if (n >= 32 && (at & 31) == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[16 * h + 2 * i], v[16 * h + 2 * i + 1]);
            st_global_256(dst + 16 * h, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
        }
    } else if (n >= 32 && (at & 15) == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(dst + 8 * q) =
                make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                           pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < n) dst[j] = __float2bfloat16_rn(v[j]);
    }
}

// Barrier of the four epilogue warps that share a half of the columns, and the same with a vote: false
// for all of them where one has given up a wait, so that none is left alone at the next barrier.
__device__ __forceinline__ void half_barrier(int half) { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); }
__device__ __forceinline__ bool half_all(int half, bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %2, 0;\n\t"
        "bar.red.and.pred q, %1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}"
        : "=r"(all)
        : "r"(1 + half), "r"(static_cast<uint32_t>(ok))
        : "memory");
    return all != 0;
}

// 64 bf16 of row `r` of a staging tile in TMA's 128-byte swizzle: 16-byte piece j lies at j ^ (r & 7).
__device__ __forceinline__ void stage_row64(unsigned char *tile, int r, int first_piece, const float (&v)[32]) {
    unsigned char *row = tile + r * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4 *>(row + (((first_piece + q) ^ (r & 7)) << 4)) =
            make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                       pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
}

template <int MODE, bool PAIR>
__global__ void __launch_bounds__(NUM_THREADS, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_out, const Args a) {
    using S = Shape<MODE, PAIR>;
    constexpr bool A_MN = MODE == kDw, B_MN = MODE == kDh || MODE == kDw;
    constexpr int BM = S::BM, STAGES = S::STAGES, A_BYTES = S::A_BYTES, STAGE_BYTES = S::STAGE_BYTES;
    constexpr smem::XentLayout L = S::layout;
    static_assert(L.stages.offset == 0 && L.stage_bytes == STAGE_BYTES, "kernel and planner disagree");
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L.full.offset);            // [STAGES] pair: used in the leader only
    uint64_t *empty = reinterpret_cast<uint64_t *>(smem + L.empty.offset);          // [STAGES] one per CTA
    uint64_t *acc_full = reinterpret_cast<uint64_t *>(smem + L.acc_full.offset);    // [2] one per CTA
    uint64_t *acc_empty = reinterpret_cast<uint64_t *>(smem + L.acc_empty.offset);  // [2] pair: used in the leader only
    uint32_t *tmem_base_slot = reinterpret_cast<uint32_t *>(smem + L.tmem_slot.offset);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_ctarank() : 0;
    const bool leader = rank == 0;
    const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, n_units = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        if (S::STORE) prefetch_tmap(&tmap_out);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * EPI_WARPS);   // the epilogue warps of every CTA
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(tmem_base_slot, 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_base_slot, 512);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();   // both CTAs' barriers exist before anyone signals across the pair
    tc_fence_after();
    const uint32_t tmem_base = *tmem_base_slot;
    pdl_launch_dependents();
    pdl_wait();

    const int counted = a.sc->count;
    const int M = MODE == kDw ? a.m : counted, N = a.n, K = MODE == kDw ? counted : a.k;
    const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
    const int tiles = tiles_m * tiles_n;
    const int splits = MODE == kDh ? a.splits : 1;
    const int k_blocks = (K + BK - 1) / BK;
    const int kb_per = (k_blocks + splits - 1) / splits;
    const int items = tiles * splits;
    struct Item {
        int tm, tn, split, kb0, nkb;
    };
    // Tiles in groups of GROUP_M tile rows, column by column inside a group, so that the units running
    // at the same time share panels in L2.  An item without K blocks (no token counts, or a short last
    // piece) has an all-zero accumulator and takes no part in the barriers.
    auto item_at = [&](int i) {
        Item it;
        it.split = i / tiles;
        const int t = i - it.split * tiles;
        const int per_group = GROUP_M * tiles_n;
        const int g = t / per_group;
        const int first_m = g * GROUP_M;
        const int in_group = min(GROUP_M, tiles_m - first_m);
        const int r = t - g * per_group;
        it.tm = first_m + r % in_group;
        it.tn = r / in_group;
        it.kb0 = it.split * kb_per;
        it.nkb = max(0, min(k_blocks, it.kb0 + kb_per) - it.kb0);
        return it;
    };
    // K blocks that go into one accumulator.  The tensor cores cut a sum off at fp32 where they add,
    // 2^-24 of the sum per 16 products on average and always towards zero: over 4096 products that
    // moved lse by 1e-5.  kLse takes the accumulator out every 1024 products and adds in registers.
    constexpr int segment = MODE == kLse ? SEGMENT : 0x7fffffff;

    if (warp == 0) {
        // ---------------- TMA producer (every CTA) ----------------
        if (lane == 0) {
            uint32_t step = 0;
            bool ok = true;
            for (int i = unit; i < items && ok; i += n_units) {
                const Item it = item_at(i);
                const int am = it.tm * BM + rank * HALF, bn = it.tn * BN + rank * HALF;
                for (int kb = it.kb0; kb < it.kb0 + it.nkb; ++kb, ++step) {
                    const int s = step % STAGES;
                    const uint32_t ph = (step / STAGES) & 1;
                    if (!mbar_wait(&empty[s], ph ^ 1, a.status, 401)) { ok = false; break; }
                    unsigned char *sa = smem + s * STAGE_BYTES, *sb = sa + A_BYTES;
                    // the leader's barrier collects the bytes of all loads of the pair
                    if (leader) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * STAGE_BYTES);
                    const uint32_t bar = PAIR ? map_to_cta(smem_u32(&full[s]), 0) : 0;
                    auto load = [&](unsigned char *dst, const CUtensorMap *map, int x, int y) {
                        if (PAIR) tma_load_2d_pair(dst, map, x, y, bar);
                        else tma_load_2d(dst, map, x, y, &full[s]);
                    };
                    if (A_MN) {
                        load(sa, &tmap_a, am, kb * BK);
                        load(sa + CHUNK_BYTES, &tmap_a, am + 64, kb * BK);
                    } else {
                        load(sa, &tmap_a, kb * BK, am);
                    }
                    constexpr int B_PARTS = B_MN ? S::B_BYTES / CHUNK_BYTES : S::B_BYTES / (HALF * BK * 2);
#pragma unroll
                    for (int c = 0; c < B_PARTS; ++c) {
                        if (B_MN) load(sb + c * CHUNK_BYTES, &tmap_b, bn + c * 64, a.b_row0 + kb * BK);
                        else load(sb + c * HALF * BK * 2, &tmap_b, kb * BK, a.b_row0 + bn + c * HALF);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader CTA only) ----------------
        if (leader && lane == 0) {
            constexpr uint32_t idesc = umma_idesc_bf16(BM, BN, B_MN, A_MN);
            // 16 K values further: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major tile
            constexpr uint64_t a_step = A_MN ? 2048 / 16 : 32 / 16, b_step = B_MN ? 2048 / 16 : 32 / 16;
            uint32_t step = 0, done = 0;
            bool ok = true;
            for (int i = unit; i < items && ok; i += n_units) {
                const Item it = item_at(i);
                for (int first = 0; first < it.nkb && ok; first += segment) {
                    const int buf = done & 1;
                    const uint32_t acc_ph = (done >> 1) & 1;
                    ++done;
                    if (!mbar_wait(&acc_empty[buf], acc_ph ^ 1, a.status, 402)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + buf * BN;
                    const int n = min(segment, it.nkb - first);
                    for (int kb = 0; kb < n; ++kb, ++step) {
                        const int s = step % STAGES;
                        const uint32_t ph = (step / STAGES) & 1;
                        if (!mbar_wait(&full[s], ph, a.status, 403)) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t sa = smem_u32(smem + s * STAGE_BYTES);
                        const uint64_t da = umma_desc_sw128(sa, A_MN ? CHUNK_BYTES : 16, 1024);
                        const uint64_t db = umma_desc_sw128(sa + A_BYTES, B_MN ? CHUNK_BYTES : 16, 1024);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            if (PAIR) umma_f16_ss_pair(d_tmem, da + k * a_step, db + k * b_step, idesc, (kb | k) != 0 ? 1u : 0u);
                            else umma_f16_ss(d_tmem, da + k * a_step, db + k * b_step, idesc, (kb | k) != 0 ? 1u : 0u);
                        }
                        if (PAIR) umma_commit_pair(&empty[s]);   // frees the slot in both CTAs
                        else umma_commit(&empty[s]);
                    }
                    if (ok) {
                        if (PAIR) umma_commit_pair(&acc_full[buf]);
                        else umma_commit(&acc_full[buf]);
                    }
                    if (segment == 0x7fffffff) break;   // (first += segment would overflow)
                }
            }
        }
    } else {
        // ---------------- epilogue (every CTA): a thread owns a row and 128 of the tile's columns ----------------
        const int lane_group = warp & 3, half = (warp - 2) >> 2;
        const bool storer = warp == 2 + 4 * half && lane == 0;   // issues the half's TMA stores
        unsigned char *stage = smem + L.out.offset + half * 2 * STORE_BYTES;
        uint32_t done = 0;
        bool ok = true;
        const float factor = MODE == kDh || MODE == kDw ? a.sc->factor : 0.0f;
        float top = -INFINITY, sum = 0.0f;
        for (int i = unit; i < items && ok; i += n_units) {
            const Item it = item_at(i);
            const int r = lane_group * 32 + lane;        // row of this CTA's half of the tile
            const int row0 = it.tm * BM + rank * HALF, row = row0 + r;
            const bool in = row < M;
            const int col0 = it.tn * BN + half * 128;    // of this piece
            int target = -1;                             // relative to col0
            float lse2 = 0.0f, g = 0.0f;
            int token = 0;
            if ((MODE == kLse || MODE == kProb) && in) target = a.target[row] - a.v0 - col0;
            if (MODE == kProb && in) {
                lse2 = static_cast<float>(static_cast<double>(a.lse[row]) * 1.4426950408889634074);
                const float largest = a.sc->largest;
                g = a.weight == nullptr ? 1.0f : largest > 0.0f ? a.weight[row] / largest : a.weight[row];
            }
            if (MODE == kDh && in && a.last) token = a.rows[row];

            int buf = 0;
            auto acquire = [&]() {
                buf = done & 1;
                const uint32_t acc_ph = (done >> 1) & 1;
                ++done;
                if (!mbar_wait(&acc_full[buf], acc_ph, a.status, 404)) ok = false;
                tc_fence_after();
            };
            auto release = [&]() {   // the accumulator is free once every CTA has drained its rows
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
                    else mbar_arrive(&acc_empty[buf]);
                }
            };
            auto columns = [&](int ch, float (&v)[32]) {
                uint32_t x[32];
                tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(lane_group * 32) << 16) +
                                  static_cast<uint32_t>(buf * BN + half * 128 + ch * 32), x);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(x[j]);
            };

            if constexpr (MODE == kLse) {
                float acc[4][32];
                for (int first = 0; first < it.nkb; first += segment) {
                    acquire();
                    if (!ok) break;
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        if (first == 0) {
                            columns(ch, acc[ch]);
                        } else {
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                uint32_t x[16];
                                tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(lane_group * 32) << 16) +
                                                  static_cast<uint32_t>(buf * BN + half * 128 + ch * 32 + q * 16), x);
                                tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < 16; ++j) acc[ch][q * 16 + j] += __uint_as_float(x[j]);
                            }
                        }
                    }
                    release();
                }
                if (!ok) break;
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    const int col = col0 + ch * 32;
                    float (&v)[32] = acc[ch];
                    const int at = target - ch * 32;   // the target's place among these 32, if it is one of them
                    if (at >= 0 && at < 32) {
                        float x = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) x = j == at ? v[j] : x;
                        a.target_logit[row] = x;
                    }
                    if (col + 32 > N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col + j >= N) v[j] = -INFINITY;
                    }
                    float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int j = 4; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], v[j]);
                    const float now = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * kLog2e);
                    const float ref = now == -INFINITY ? 0.0f : now;   // every logit so far is -inf
                    float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 32; ++j) s4[j & 3] += ex2(fmaf(v[j], kLog2e, -ref));
                    sum = sum * ex2(top - ref) + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
                    top = now;
                }
                // one slot per tile and half, or (a.running: a single tile row) one per unit and half
                if (!a.running || i + n_units >= items) {
                    const int slot = a.part0 + (a.running ? unit * 2 : it.tn * 2) + half;
                    if (in && (a.running || col0 < N)) a.partial[slot * a.ld_partial + row] = make_float2(top, sum);
                    top = -INFINITY;
                    sum = 0.0f;
                }
            } else {
                const bool tma = S::STORE && a.tma_out;
                if (it.nkb) acquire();
                if (tma) ok = half_all(half, ok);
                if (!ok) break;
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {   // 64 columns
                    const int col = col0 + part * 64;
                    unsigned char *tile = stage + part * STORE_BYTES;
                    if (tma) {
                        // the store of the previous tile's same part has left this staging tile
                        if (storer) tma_store_wait_read<1>();
                        half_barrier(half);
                    }
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const int ch = part * 2 + sub, c = col + sub * 32;
                        float v[32];
                        if (it.nkb) {
                            columns(ch, v);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.0f;
                        }
                        if (ch == 3 && it.nkb) release();
                        if (MODE == kProb) {
                            const int at = target - ch * 32;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                float p = ex2(fmaf(v[j], kLog2e, -lse2));
                                if (j == at) p -= 1.0f;
                                v[j] = in ? p * g : 0.0f;
                            }
                        }
                        if (MODE == kDw) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= factor;
                        }
                        if (S::STORE) {
                            if (tma) stage_row64(tile, r, sub * 4, v);
                            else if (in && c < N) store_row32(a.out + static_cast<int64_t>(row) * a.ldo + c, v, N - c);
                        }
                        if (MODE == kDh && in && c < N) {
                            float *s = a.slab + it.split * a.slab_stride + static_cast<int64_t>(row) * a.ld_slab + c;
                            if (!a.first) {
#pragma unroll
                                for (int j = 0; j < 32; j += 4) {
                                    const float4 o = *reinterpret_cast<const float4 *>(s + j);
                                    v[j] += o.x;
                                    v[j + 1] += o.y;
                                    v[j + 2] += o.z;
                                    v[j + 3] += o.w;
                                }
                            }
                            if (a.last) {
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] *= factor;
                                store_row32(a.out + static_cast<int64_t>(token) * a.ldo + c, v, N - c);
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    *reinterpret_cast<float4 *>(s + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                            }
                        }
                    }
                    if (tma) {
                        fence_proxy_async_smem();
                        half_barrier(half);
                        if (storer) {
                            // rows behind the matrix and columns behind its last are cut off by the tensor map
                            if (col < N) tma_store_2d(&tmap_out, tile, col, row0);
                            tma_store_commit();
                        }
                    }
                }
            }
        }
        if (S::STORE && storer) tma_store_wait_all<0>();
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();   // no CTA may leave while its partner can still signal into it
    if (warp == 1) {
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

// Lists the tokens that count, in their order: one block, 1024 tokens a step.
struct PrepareArgs {
    const int64_t *targets;
    int T, V;
    int64_t ignore;
    const float *lse;       // backward: per token
    const float *dloss;     // backward: per token, or NULL for the mean
    const float *total;     // backward, mean: total[1] tokens count
    float scale;
    int *rows, *target;     // [T]
    float *lse_c, *weight_c;
    Scalars *sc;
    float *loss_out, *lse_out;   // forward: values of the tokens that do not count
};

__global__ void __launch_bounds__(1024) xent_prepare_kernel(const PrepareArgs a) {
    __shared__ int counts[32];
    __shared__ int bads[32];
    __shared__ float tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    int running = 0, bad_here = 0;
    float top = 0.0f;
    for (int64_t base = 0; base < a.T; base += 1024) {
        const int64_t i = base + threadIdx.x;
        const bool in = i < a.T;
        const int64_t t = in ? a.targets[i] : a.ignore;
        const bool keep = in && t != a.ignore && t >= 0 && t < a.V;
        const bool bad = in && t != a.ignore && !keep;
        bad_here += bad;
        const unsigned votes = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) counts[wid] = __popc(votes);
        __syncthreads();
        int before = 0, all = 0;
        {
            const int c = counts[lane];
            int incl = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            before = __shfl_sync(0xffffffffu, incl - c, wid);
            all = __shfl_sync(0xffffffffu, incl, 31);
        }
        if (keep) {
            const int at = running + before + __popc(votes & ((1u << lane) - 1));
            a.rows[at] = (int)i;
            a.target[at] = (int)t;
            if (a.lse) a.lse_c[at] = a.lse[i];
            if (a.dloss) {
                const float g = a.dloss[i];
                a.weight_c[at] = g;
                top = fmaxf(top, fabsf(g));
            }
        } else if (in) {
            if (a.loss_out) a.loss_out[i] = bad ? __int_as_float(0x7fffffff) : 0.0f;
            if (a.lse_out) a.lse_out[i] = bad ? __int_as_float(0x7fffffff) : 0.0f;
        }
        running += all;
        __syncthreads();
    }
    top = warp_max(top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bad_here += __shfl_xor_sync(0xffffffffu, bad_here, o);
    if (lane == 0) {
        tops[wid] = top;
        bads[wid] = bad_here;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) {
            top = fmaxf(top, tops[w]);
            bad_here += bads[w];
        }
        Scalars s;
        s.count = running;
        s.bad = bad_here;
        s.largest = top;
        // all weights 0 (or NaN, which the maximum passes over): G takes them as they are
        s.factor = running == 0 ? 0.0f : a.dloss ? (top > 0.0f ? a.scale * top : a.scale) : a.total ? a.scale / a.total[1] : 0.0f;
        *a.sc = s;
    }
}

// Packs the rows of the tokens that count, a block per row, and zeroes the rows behind them up to a
// multiple of 64 (they are K rows of dW's product); backward: zeroes dH of the tokens that do not count.
__global__ void __launch_bounds__(128)
xent_pack_rows_kernel(const __nv_bfloat16 *H, int64_t ldh, int D, __nv_bfloat16 *Hc, int64_t ldc, const int *rows, const Scalars *sc,
                      const int64_t *targets, int64_t ignore, int T, int V, __nv_bfloat16 *dH, int64_t lddh) {
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x;
    const int count = sc->count;
    __nv_bfloat16 *dst = Hc + r * ldc;
    if (r < count) {
        const __nv_bfloat16 *src = H + rows[r] * ldh;
        if ((reinterpret_cast<uintptr_t>(H) & 15) == 0 && ldh % 8 == 0) {
            for (int j = threadIdx.x; j < D / 8; j += 128)
                reinterpret_cast<uint4 *>(dst)[j] = __ldcs(reinterpret_cast<const uint4 *>(src) + j);
            for (int j = D / 8 * 8 + threadIdx.x; j < D; j += 128) dst[j] = src[j];
        } else {
            for (int j = threadIdx.x; j < D; j += 128) dst[j] = src[j];
        }
    } else if (r < (count + BK - 1) / BK * BK) {
        for (int j = threadIdx.x; j < ldc / 8; j += 128) reinterpret_cast<uint4 *>(dst)[j] = make_uint4(0, 0, 0, 0);
    }
    if (dH && r < T) {
        const int64_t t = targets[r];
        if (t == ignore || t < 0 || t >= V)
            for (int j = threadIdx.x; j < D; j += 128) dH[r * lddh + j] = __float2bfloat16_rn(0.0f);
    }
}

// Rows of W whose pitch or address TMA cannot take, packed to a pitch of 16 bytes' multiple.
__global__ void __launch_bounds__(128)
xent_pack_weight_kernel(const __nv_bfloat16 *W, int64_t ldw, int D, __nv_bfloat16 *Wc, int64_t ldc) {
    pdl_launch_dependents();
    pdl_wait();
    const __nv_bfloat16 *src = W + static_cast<int64_t>(blockIdx.x) * ldw;
    __nv_bfloat16 *dst = Wc + static_cast<int64_t>(blockIdx.x) * ldc;
    for (int j = threadIdx.x; j < D; j += 128) dst[j] = src[j];
}

// Joins the tile columns' maxima and sums: 32 rows per block, 32 threads deep.  The last block to
// finish adds up the blocks' sums of losses, in their order.
__global__ void __launch_bounds__(1024)
xent_finish_kernel(const float2 *partial, int64_t ld_partial, int parts, const float *target_logit, const int *rows,
                   const Scalars *sc, float *loss, float *lse, float *total, double *block_sums, unsigned int *ticket) {
    __shared__ float tops[32][33], sums[32][33];
    __shared__ bool last_block;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, deep = threadIdx.x >> 5;
    const int count = sc->count;
    const int row = blockIdx.x * 32 + lane;
    float top = -INFINITY, sum = 0.0f;
    auto join = [&](float m, float s) {
        const float now = fmaxf(top, m);
        const float ref = now == -INFINITY ? 0.0f : now;
        sum = sum * ex2(top - ref) + s * ex2(m - ref);
        top = now;
    };
    if (row < count) {
#pragma unroll 4
        for (int p = deep; p < parts; p += 32) {
            const float2 v = partial[p * ld_partial + row];
            join(v.x, v.y);
        }
    }
    tops[deep][lane] = top;
    sums[deep][lane] = sum;
    __syncthreads();
    if (deep == 0) {
        double mine = 0.0;
        if (row < count) {
            top = -INFINITY;
            sum = 0.0f;
#pragma unroll
            for (int d = 0; d < 32; ++d) join(tops[d][lane], sums[d][lane]);
            const double l = static_cast<double>(top) * kLn2 + log(static_cast<double>(sum));
            const double x = l - static_cast<double>(target_logit[row]);
            const int token = rows[row];
            if (lse) lse[token] = static_cast<float>(l);
            if (loss) loss[token] = static_cast<float>(x);
            mine = x;
        }
        if (total) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
            if (lane == 0) {
                block_sums[blockIdx.x] = mine;
                __threadfence();
                last_block = atomicAdd(ticket, 1u) == gridDim.x - 1;
            }
        } else if (lane == 0) {
            last_block = false;
        }
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    __shared__ double deep_sums[32];
    double all = 0.0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += 1024) all += __ldcg(block_sums + b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) deep_sums[deep] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        all = 0.0;
        for (int d = 0; d < 32; ++d) all += deep_sums[d];
        total[0] = sc->bad ? __int_as_float(0x7fffffff) : static_cast<float>(all);
        total[1] = static_cast<float>(count);
        *ticket = 0;
    }
}

// dH of split sums: one block per packed row.
__global__ void __launch_bounds__(128)
xent_dh_finish_kernel(const float *slab, int64_t slab_stride, int64_t ld_slab, int splits, const int *rows, const Scalars *sc,
                      int D, __nv_bfloat16 *dH, int64_t lddh) {
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x >= sc->count) return;
    const float factor = sc->factor;
    __nv_bfloat16 *dst = dH + rows[blockIdx.x] * lddh;
    const float *src = slab + blockIdx.x * ld_slab;
    for (int j = threadIdx.x; j < D; j += 128) {
        float s = 0.0f;
        for (int k = 0; k < splits; ++k) s += src[k * slab_stride + j];
        dst[j] = __float2bfloat16_rn(s * factor);
    }
}

// ---- host side -----------------------------------------------------------------------------------

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Scratch {   // hands out aligned pieces; a first walk with base NULL measures
    unsigned char *base = nullptr;
    size_t used = 0;
    template <typename T>
    T *take(int64_t n) {
        T *p = reinterpret_cast<T *>(base + used);
        used += (size_t)up(n * (int64_t)sizeof(T), 1024);
        return p;
    }
};

struct Call {
    gb200_ctx *ctx;
    const __nv_bfloat16 *H, *W;
    int64_t ldh, ldw;
    const int64_t *targets;
    int T, V, D;
    int64_t ignore;
    cudaStream_t stream;

    bool pack_w() const { return (reinterpret_cast<uintptr_t>(W) & 15) != 0 || ldw % 8 != 0; }
    int64_t dp() const { return up(D, 8); }
    int tiles(int64_t n) const { return (int)((n + 255) / 256); }
};

int map_of(gb200_ctx *ctx, const void *p, int64_t cols, int64_t rows, int64_t ld, bool mn_major, CUtensorMap *out) {
    return get_tmap_2d(ctx, p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)cols, (uint64_t)rows, (uint64_t)ld * 2, 64,
                       mn_major ? BK : HALF, CU_TENSOR_MAP_SWIZZLE_128B, out);
}

// With at most 128 tokens on one CTA per tile, else on pairs; dW's rows are classes, always on pairs.
bool on_pairs(const Call &c, int mode) { return mode == kDw || c.T > 128; }
int units(const Call &c, int mode) { return std::max(on_pairs(c, mode) ? c.ctx->sm_count / 2 : c.ctx->sm_count, 1); }
int64_t tile_rows(const Call &c, int mode, int64_t rows) {
    const int bm = on_pairs(c, mode) ? 256 : 128;
    return (rows + bm - 1) / bm;
}

template <int MODE, bool PAIR>
int launch_as(const Call &c, const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &to, int64_t n_units, const Args &a) {
    constexpr int bytes = Shape<MODE, PAIR>::layout.dynamic_bytes;
    auto kern = xent_gemm_kernel<MODE, PAIR>;
    const int rc = ensure_dynamic_smem(c.ctx, kern, bytes);
    if (rc) return rc;
    GB200_CUDA_TRY(launch_pdl_cluster(kern, dim3((unsigned)(n_units * (PAIR ? 2 : 1))), dim3(NUM_THREADS), (size_t)bytes, c.stream,
                                      PAIR ? 2u : 1u, ta, tb, to, a));
    static const char *const names[] = {"xent_gemm_kernel<lse>", "xent_gemm_kernel<prob>", "xent_gemm_kernel<dh>",
                                        "xent_gemm_kernel<dw>"};
    return after_launch(c.ctx, names[MODE]);
}

// Returns the number of units launched (CTAs or pairs) through *used.
template <int MODE>
int launch(const Call &c, const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &to, int64_t items, Args a, int *used = nullptr) {
    const int64_t n = std::min<int64_t>(units(c, MODE), items);
    if (used) *used = (int)n;
    a.status = c.ctx->d_status;
    if constexpr (MODE != kDw)
        if (!on_pairs(c, MODE)) return launch_as<MODE, false>(c, ta, tb, to, n, a);
    return launch_as<MODE, true>(c, ta, tb, to, n, a);
}

int prepare(const Call &c, const PrepareArgs &p) {
    GB200_CUDA_TRY(launch_pdl(xent_prepare_kernel, dim3(1), dim3(1024), 0, c.stream, p));
    return after_launch(c.ctx, "xent_prepare_kernel");
}

int pack_rows(const Call &c, __nv_bfloat16 *Hc, const int *rows, const Scalars *sc, __nv_bfloat16 *dH, int64_t lddh) {
    GB200_CUDA_TRY(launch_pdl(xent_pack_rows_kernel, dim3((unsigned)up(c.T, BK)), dim3(128), 0, c.stream, c.H, c.ldh, c.D, Hc,
                              c.dp(), rows, sc, c.targets, c.ignore, c.T, c.V, dH, lddh));
    return after_launch(c.ctx, "xent_pack_rows_kernel");
}

int pack_weight(const Call &c, int64_t v0, int64_t rows, __nv_bfloat16 *Wc) {
    GB200_CUDA_TRY(launch_pdl(xent_pack_weight_kernel, dim3((unsigned)rows), dim3(128), 0, c.stream, c.W + v0 * c.ldw, c.ldw, c.D,
                              Wc, c.dp()));
    return after_launch(c.ctx, "xent_pack_weight_kernel");
}

int forward(const Call &c, float *loss, float *lse, float *total) {
    // the whole vocabulary at once, unless W has to be packed first
    const int64_t piece = c.pack_w() ? std::min<int64_t>(c.V, std::max<int64_t>(kPieceBytes / (c.dp() * 2) / 256 * 256, 256)) : c.V;
    // one row of tiles: a slot per unit and piece, else one per tile column; both times two halves
    const bool running = tile_rows(c, kLse, c.T) == 1;
    const int64_t pieces = (c.V + piece - 1) / piece;
    const int64_t parts = 2 * (running ? units(c, kLse) * pieces : c.tiles(c.V) + pieces);
    Scratch s;
    int *rows, *target;
    Scalars *sc;
    float *target_logit;
    float2 *partial;
    double *block_sums;
    __nv_bfloat16 *Hc, *Wc;
    for (int pass = 0; pass < 2; ++pass) {
        s.used = 0;
        sc = s.take<Scalars>(1);
        rows = s.take<int>(c.T);
        target = s.take<int>(c.T);
        target_logit = s.take<float>(c.T);
        block_sums = s.take<double>((c.T + 31) / 32);
        partial = s.take<float2>(parts * c.T);
        Hc = s.take<__nv_bfloat16>(up(c.T, BK) * c.dp());
        Wc = c.pack_w() ? s.take<__nv_bfloat16>(piece * c.dp()) : nullptr;
        if (pass == 0) {
            void *base = nullptr;
            const int rc = scratch_reserve(c.ctx, s.used, c.stream, &base);
            if (rc) return rc;
            s.base = static_cast<unsigned char *>(base);
        }
    }
    PrepareArgs p{};
    p.targets = c.targets;
    p.T = c.T;
    p.V = c.V;
    p.ignore = c.ignore;
    p.rows = rows;
    p.target = target;
    p.sc = sc;
    p.loss_out = loss;
    p.lse_out = lse;
    int rc = prepare(c, p);
    if (rc) return rc;
    rc = pack_rows(c, Hc, rows, sc, nullptr, 0);
    if (rc) return rc;
    CUtensorMap ta, tb;
    rc = map_of(c.ctx, Hc, c.D, c.T, c.dp(), false, &ta);
    if (rc) return rc;
    int part = 0;
    for (int64_t v0 = 0; v0 < c.V; v0 += piece) {
        const int64_t n = std::min<int64_t>(piece, c.V - v0);
        if (c.pack_w()) {
            rc = pack_weight(c, v0, n, Wc);
            if (rc) return rc;
        }
        rc = c.pack_w() ? map_of(c.ctx, Wc, c.D, n, c.dp(), false, &tb) : map_of(c.ctx, c.W, c.D, c.V, c.ldw, false, &tb);
        if (rc) return rc;
        Args a{};
        a.sc = sc;
        a.n = (int)n;
        a.k = c.D;
        a.b_row0 = c.pack_w() ? 0 : (int)v0;
        a.v0 = (int)v0;
        a.target = target;
        a.partial = partial;
        a.ld_partial = c.T;
        a.part0 = part;
        a.target_logit = target_logit;
        a.running = running;
        int used = 0;
        rc = launch<kLse>(c, ta, tb, tb, tile_rows(c, kLse, c.T) * c.tiles(n), a, &used);
        if (rc) return rc;
        part += running ? 2 * used : (int)((n + 127) / 128);   // whole tiles (pieces are multiples of 256) but for the last
    }
    GB200_CUDA_TRY(launch_pdl(xent_finish_kernel, dim3((unsigned)((c.T + 31) / 32)), dim3(1024), 0, c.stream, partial, (int64_t)c.T,
                              part, target_logit, rows, sc, loss, lse, total, block_sums, c.ctx->tickets + kTicketXent));
    return after_launch(c.ctx, "xent_finish_kernel");
}

// Ranges that the K dimension of dH's product is cut into so that its tiles fill the SMs: rounds
// of (tile, range) items times a range's K blocks, each item charged 8 blocks for its epilogue.
int pick_splits(int64_t tiles, int64_t k_blocks, int64_t units, int64_t slab_bytes) {
    int best = 1;
    int64_t best_cost = INT64_MAX;
    for (int s = 1; s <= 64 && s <= k_blocks && (s == 1 || s * slab_bytes <= kSlabBytes); ++s) {
        const int64_t cost = ((tiles * s + units - 1) / units) * ((k_blocks + s - 1) / s + 8) + (s > 1 ? 16 : 0);
        if (cost < best_cost) {
            best_cost = cost;
            best = s;
        }
    }
    return best;
}

int backward(const Call &c, const float *lse, const float *dloss, const float *total, float scale, __nv_bfloat16 *dH, int64_t lddh,
             __nv_bfloat16 *dW, int64_t lddw) {
    int64_t piece = std::max<int64_t>(kPieceBytes / (2ll * c.T) / 256 * 256, 256);
    if (c.pack_w()) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (c.dp() * 2) / 256 * 256, 256));
    piece = std::min<int64_t>(piece, c.V);
    const int64_t ld_slab = up(c.D, 32), slab_stride = ld_slab * c.T, ldg = up(piece, 64);
    const int64_t dh_tiles = tile_rows(c, kDh, c.T) * c.tiles(c.D);
    const int splits = pick_splits(dh_tiles, up(piece, BK) / BK, units(c, kDh), slab_stride * 4);
    const bool slab_wanted = dH && (splits > 1 || piece < c.V);
    Scratch s;
    int *rows, *target;
    Scalars *sc;
    float *lse_c, *weight_c, *slab;
    __nv_bfloat16 *Hc, *Wc, *G;
    for (int pass = 0; pass < 2; ++pass) {
        s.used = 0;
        sc = s.take<Scalars>(1);
        rows = s.take<int>(c.T);
        target = s.take<int>(c.T);
        lse_c = s.take<float>(c.T);
        weight_c = s.take<float>(c.T);
        Hc = s.take<__nv_bfloat16>(up(c.T, BK) * c.dp());
        Wc = c.pack_w() ? s.take<__nv_bfloat16>(piece * c.dp()) : nullptr;
        G = s.take<__nv_bfloat16>(up(c.T, 256) * ldg);
        slab = slab_wanted ? s.take<float>(splits * slab_stride) : nullptr;
        if (pass == 0) {
            void *base = nullptr;
            const int rc = scratch_reserve(c.ctx, s.used, c.stream, &base);
            if (rc) return rc;
            s.base = static_cast<unsigned char *>(base);
        }
    }
    PrepareArgs p{};
    p.targets = c.targets;
    p.T = c.T;
    p.V = c.V;
    p.ignore = c.ignore;
    p.lse = lse;
    p.dloss = dloss;
    p.total = total;
    p.scale = scale;
    p.rows = rows;
    p.target = target;
    p.lse_c = lse_c;
    p.weight_c = weight_c;
    p.sc = sc;
    int rc = prepare(c, p);
    if (rc) return rc;
    rc = pack_rows(c, Hc, rows, sc, dH, lddh);
    if (rc) return rc;
    CUtensorMap h_k, h_mn;
    rc = map_of(c.ctx, Hc, c.D, up(c.T, BK), c.dp(), false, &h_k);
    if (!rc) rc = map_of(c.ctx, Hc, c.D, up(c.T, BK), c.dp(), true, &h_mn);
    if (rc) return rc;
    for (int64_t v0 = 0; v0 < c.V; v0 += piece) {
        const int64_t n = std::min<int64_t>(piece, c.V - v0);
        const bool last = v0 + n == c.V;
        if (c.pack_w()) {
            rc = pack_weight(c, v0, n, Wc);
            if (rc) return rc;
        }
        CUtensorMap w_k, w_mn, g_k, g_mn;
        const void *wp = c.pack_w() ? static_cast<const void *>(Wc) : c.W;
        const int64_t w_rows = c.pack_w() ? n : c.V, w_ld = c.pack_w() ? c.dp() : c.ldw;
        rc = map_of(c.ctx, wp, c.D, w_rows, w_ld, false, &w_k);
        if (!rc) rc = map_of(c.ctx, wp, c.D, w_rows, w_ld, true, &w_mn);
        if (!rc) rc = map_of(c.ctx, G, n, up(c.T, 256), ldg, false, &g_k);
        if (!rc) rc = map_of(c.ctx, G, n, up(c.T, 256), ldg, true, &g_mn);
        if (rc) return rc;
        Args a{};
        a.sc = sc;
        a.b_row0 = c.pack_w() ? 0 : (int)v0;
        a.v0 = (int)v0;
        a.target = target;
        a.rows = rows;
        a.n = (int)n;
        a.k = c.D;
        a.lse = lse_c;
        a.weight = dloss ? weight_c : nullptr;
        a.out = G;
        a.ldo = ldg;
        a.tma_out = 1;
        rc = launch<kProb>(c, h_k, w_k, g_k, tile_rows(c, kProb, c.T) * c.tiles(n), a);
        if (rc) return rc;
        if (dH) {
            Args d = a;
            d.n = c.D;
            d.k = (int)n;
            d.slab = slab;
            d.slab_stride = slab_stride;
            d.ld_slab = ld_slab;
            d.splits = splits;
            d.first = v0 == 0;
            d.last = last && splits == 1;
            d.out = dH;
            d.ldo = lddh;
            rc = launch<kDh>(c, g_k, w_mn, g_k, dh_tiles * splits, d);
            if (rc) return rc;
        }
        if (dW) {
            Args d = a;
            d.m = (int)n;
            d.n = c.D;
            d.b_row0 = 0;   // B is the packed H here
            d.out = dW + v0 * lddw;
            d.ldo = lddw;
            d.tma_out = (reinterpret_cast<uintptr_t>(d.out) & 15) == 0 && lddw % 8 == 0;
            CUtensorMap out = g_k;
            if (d.tma_out) {
                rc = map_of(c.ctx, d.out, c.D, n, lddw, false, &out);
                if (rc) return rc;
            }
            rc = launch<kDw>(c, g_mn, h_mn, out, (int64_t)c.tiles(n) * c.tiles(c.D), d);
            if (rc) return rc;
        }
    }
    if (dH && splits > 1) {
        GB200_CUDA_TRY(launch_pdl(xent_dh_finish_kernel, dim3((unsigned)c.T), dim3(128), 0, c.stream, slab, slab_stride, ld_slab,
                                  splits, rows, sc, c.D, dH, lddh));
        return after_launch(c.ctx, "xent_dh_finish_kernel");
    }
    return GB200_OK;
}

int check(const void *H, int64_t ldh, const void *W, int64_t ldw, const int64_t *targets, int64_t T, int64_t V, int64_t D) {
    GB200_REQUIRE(T >= 0 && V >= 0 && D >= 0, GB200_ERR_INVALID_ARG, "negative extent");
    GB200_REQUIRE(T <= (1 << 26) && V <= (1 << 26) && D <= (1 << 20), GB200_ERR_TOO_LARGE,
                  "more than 2^26 tokens or classes, or rows of more than 2^20 elements");
    GB200_REQUIRE(V > 0 && D > 0, GB200_ERR_INVALID_ARG, "no classes, or rows without elements");
    GB200_REQUIRE(W != nullptr && (T == 0 || (H != nullptr && targets != nullptr)), GB200_ERR_INVALID_ARG, "NULL operand");
    GB200_REQUIRE(ldw >= D && (T <= 1 || ldh >= D), GB200_ERR_INVALID_ARG, "leading dimension smaller than the row");
    GB200_REQUIRE(((reinterpret_cast<uintptr_t>(H) | reinterpret_cast<uintptr_t>(W)) & 1) == 0 &&
                      (reinterpret_cast<uintptr_t>(targets) & 7) == 0,
                  GB200_ERR_INVALID_ARG, "pointer not aligned to its element");
    return GB200_OK;
}

}  // namespace
}  // namespace gb200

using namespace gb200;

extern "C" {

int gb200_linear_xent_bf16(gb200_ctx *ctx, const void *H, int64_t ldh, const void *W, int64_t ldw, const int64_t *targets,
                           int64_t T, int64_t V, int64_t D, int64_t ignore_index, float *loss, float *lse, float *total,
                           void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check(H, ldh, W, ldw, targets, T, V, D);
    if (rc) return rc;
    GB200_REQUIRE(loss || lse || total, GB200_ERR_INVALID_ARG, "nothing to produce: loss, lse and total are NULL");
    GB200_REQUIRE(((reinterpret_cast<uintptr_t>(loss) | reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(total)) & 3) == 0,
                  GB200_ERR_INVALID_ARG, "pointer not aligned to its element");
    const Range in[3] = {Range(H, ldh, T, D, 2), Range(W, ldw, V, D, 2), Range(targets, T, 1, T, 8)};
    const Range out[3] = {Range(loss, T, 1, T, 4), Range(lse, T, 1, T, 4), Range(total, 2, 1, 2, 4)};
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j)
            GB200_REQUIRE(!out[i].overlaps(in[j]) && (i == j || !out[i].overlaps(out[j])), GB200_ERR_INVALID_ARG,
                          "an output overlaps another operand");
    DeviceScope scope;
    rc = scope.enter(ctx);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        if (total) GB200_CUDA_TRY(cudaMemsetAsync(total, 0, 2 * sizeof(float), st));
        return GB200_OK;
    }
    const Call c{ctx, static_cast<const __nv_bfloat16 *>(H), static_cast<const __nv_bfloat16 *>(W), ldh, ldw, targets, (int)T,
                 (int)V, (int)D, ignore_index, st};
    return forward(c, loss, lse, total);
}

int gb200_linear_xent_bf16_backward(gb200_ctx *ctx, const void *H, int64_t ldh, const void *W, int64_t ldw,
                                    const int64_t *targets, const float *lse, const float *dloss, const float *total,
                                    int64_t T, int64_t V, int64_t D, int64_t ignore_index, float scale, void *dH,
                                    int64_t lddh, void *dW, int64_t lddw, void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check(H, ldh, W, ldw, targets, T, V, D);
    if (rc) return rc;
    GB200_REQUIRE(dH || dW, GB200_ERR_INVALID_ARG, "nothing to produce: dH and dW are NULL");
    GB200_REQUIRE((dloss != nullptr) != (total != nullptr), GB200_ERR_INVALID_ARG,
                  "either dloss (a weight per token) or total (the mean) is wanted");
    GB200_REQUIRE(T == 0 || lse != nullptr, GB200_ERR_INVALID_ARG, "lse is NULL");
    GB200_REQUIRE((!dH || T <= 1 || lddh >= D) && (!dW || lddw >= D), GB200_ERR_INVALID_ARG, "leading dimension smaller than the row");
    GB200_REQUIRE(((reinterpret_cast<uintptr_t>(dH) | reinterpret_cast<uintptr_t>(dW)) & 1) == 0 &&
                      ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(dloss) | reinterpret_cast<uintptr_t>(total)) & 3) == 0,
                  GB200_ERR_INVALID_ARG, "pointer not aligned to its element");
    const Range in[6] = {Range(H, ldh, T, D, 2),       Range(W, ldw, V, D, 2),       Range(targets, T, 1, T, 8),
                         Range(lse, T, 1, T, 4),       Range(dloss, T, 1, T, 4),     Range(total, 2, 1, 2, 4)};
    const Range rdh(dH, lddh, T, D, 2), rdw(dW, lddw, V, D, 2);
    for (const Range &r : in)
        GB200_REQUIRE(!r.overlaps(rdh) && !r.overlaps(rdw), GB200_ERR_INVALID_ARG, "an output overlaps another operand");
    GB200_REQUIRE(!rdh.overlaps(rdw), GB200_ERR_INVALID_ARG, "an output overlaps another operand");
    DeviceScope scope;
    rc = scope.enter(ctx);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        if (dW) GB200_CUDA_TRY(cudaMemset2DAsync(dW, lddw * 2, 0, D * 2, V, st));
        return GB200_OK;
    }
    const Call c{ctx, static_cast<const __nv_bfloat16 *>(H), static_cast<const __nv_bfloat16 *>(W), ldh, ldw, targets, (int)T,
                 (int)V, (int)D, ignore_index, st};
    return backward(c, lse, dloss, total, scale, static_cast<__nv_bfloat16 *>(dH), lddh, static_cast<__nv_bfloat16 *>(dW), lddw);
}

}  // extern "C"
