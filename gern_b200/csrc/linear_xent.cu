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
// with few tokens the reading of W.  All four products run in one kernel template (TMA ring, one thread
// issuing tcgen05.mma, two accumulators in TMEM; the structure of gemm_bf16_2cta.cu, on pairs of CTAs or, with
// few tokens, on single ones: see Tiling), which differs from that one in its epilogues and in operands
// that are read with the MN dimension contiguous: W as the K x N operand of dH, G as the M x K operand and
// H as the K x N operand of dW.  No operand is ever transposed in memory.  Measured, 8192 x 131072 x 4096:
// loss 5.5 ms from a cool start (1600 TFLOP/s), 6.1-6.4 ms under the power cap; both gradients 20.2-20.7 ms
// (1275-1305 TFLOP/s, always under the cap, where cuBLAS holds 1398 on one square product).
//
// Only tokens that count take part: their rows of H are packed first (T x D x 4 bytes of traffic, 0.1 % of
// the products' time at that size).  Ignored tokens then cost nothing, and what their rows hold (NaN,
// infinities) reaches no gradient; a product with zeros in G would spread it.  The number of counted
// tokens stays on the device: kernels read it and take that many rows of tiles.
//
// G goes through memory in pieces of the vocabulary (kPieceBytes), as bf16.  That rounding is half a
// step, 2^-8 relative at most, independent from entry to entry; the factor that all tokens share (the
// largest finite |g_t|) is kept out of it and applied to the fp32 sums, since a common factor's rounding
// would not average out: the entry at the target, near -g_t, would be off by the same share everywhere.
#include <algorithm>
#include <math.h>

#include "common.cuh"
#include "smem_plan.hpp"

namespace gb200 {
namespace {

constexpr int BN = 256, BK = 64, HALF = 128;
constexpr int CHUNK_BYTES = 64 * BK * 2;    // MN-major operand: 64 columns x 64 K rows, 128 bytes per row
constexpr int kFewT = 32;                   // tokens of the kFew tiling
constexpr int GROUP_M = 8;                  // tile rows per rasterisation group
constexpr int EPI_WARPS = 8;                // two per quarter of the TMEM lanes, 128 columns each
constexpr int NUM_THREADS = 64 + 32 * EPI_WARPS;
constexpr int STORE_BYTES = 32 * 64 * 2;    // staging tile of a TMA store: a warp's 32 rows x 64 columns

// kLse: running maxima and sums of the logits.  kProb: G.  kGrad: the tiles of dH, then those of dW.
enum Mode { kLse, kProb, kGrad };

// K blocks that the tensor cores add up before the accumulator is taken out.  They cut a sum off at fp32 where they
// add, 2^-24 of the sum per 16 products on average and always towards zero: over 4096 products that moved lse by
// 1e-5.  kLse leaves the accumulator every 1024 products and adds in registers.  G is rounded to bf16, 2^-8, which 256
// such steps in a logit (kProb, 4096 products: 2^-16 of it) do not reach, and neither do 1024 steps (kGrad, 16384
// products: 2^-14) in the gradients; left to go on, 2^22 tokens of one sign made dW 2.6 % short.  Longer sums of
// these two are kept in the other accumulator, to which the epilogue adds while the MMA waits (gradients of 32768
// tokens over 32768 x 2048, two segments: 10.8 ms, 11.1 without them, 11.5 with sums in registers, which spill).
constexpr int kSumBlocks[] = {16, 64, 256};

// How the tokens' tiles lie on the machine.
// kPairs: 256 x 256 tiles on two CTAs, each of which stages its half of A and of B.
// kSingles: tiles of 128 rows on one CTA, where pairs would spend their MMA time on rows that do not exist
// (65536 x 4096, one token: tensor pipe 74 % active at 58 % of the DRAM rate, 126 us; on single CTAs 106 us).
// kFew: at most 32 tokens.  Only their rows are loaded, and the room goes to more stages: what bounds
// the reading of W is bytes in flight (the same, four stages 106, six 92 us).  The MMA's other 96 rows are
// whatever lies behind the 32 in shared memory, and their results are never looked at.
enum Tiling { kPairs, kSingles, kFew };
template <int MODE, int TILING>
struct Shape {
    static constexpr bool PAIR = TILING == kPairs;
    static constexpr bool STORE = MODE != kLse;      // results leave through shared memory
    static constexpr int BM = PAIR ? 256 : 128;
    static constexpr int A_ROWS = TILING == kFew && MODE != kGrad ? kFewT : HALF;
    static constexpr int A_BYTES = A_ROWS * BK * 2, B_BYTES = (PAIR ? HALF : BN) * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = A_ROWS == kFewT ? (STORE ? 5 : 6) : PAIR ? (STORE ? 5 : 6) : 4;
    static constexpr int OUT_BUFFERS = PAIR ? 2 : 1;      // staging tiles per epilogue warp
    static constexpr smem::XentLayout layout =
        smem::xent_layout(STAGES, STAGE_BYTES, STORE ? EPI_WARPS * OUT_BUFFERS * STORE_BYTES : 128 * 8);
    static_assert(layout.dynamic_bytes <= smem::kMaxDynamicBytes, "the ring exceeds a block's shared memory");
};

// G of one piece of the vocabulary: large enough that a piece fills the SMs many times over, small
// beside W and dW (1 GiB each at 131072 x 4096).  A piece has 2048 classes at least, however many the
// tokens: every piece adds to dH in fp32, and with fewer classes that traffic would bound it.
constexpr int64_t kPieceBytes = 256ll << 20, kPieceClasses = 2048;
constexpr int64_t kSlabBytes = 512ll << 20;   // most that split sums of dH may take

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;

// What the first kernel leaves for the others.
struct Scalars {
    int count;        // tokens that count
    int bad;          // tokens whose target is neither in [0, V) nor ignore_index
    float factor;     // common factor of the gradients
    float largest;    // largest finite |g_t| where `factor` holds it, 0 where G takes the weights as they are
};

struct Args {
    const Scalars *sc;
    int bn;                    // columns per tile; kPairs and kGrad: BN
    int n, k;                  // kLse, kProb: classes of this piece, D.  kGrad: D, classes of this piece
    int w_row0;                // row of W's tensor map where this piece starts
    int v0;                    // first class of this piece
    const int *target;         // [count]
    // kLse
    float2 *partial;           // maximum (times log2 e) and sum: [slot][row], or (running) [row][slot]
    int64_t ld_partial;
    int part0;                 // first slot of this piece
    int running;               // one row of tiles: a unit keeps its maximum and sum over all its tiles
    int finish;                // running: the last CTA of this launch joins the slots
    float *target_logit;       // [count]
    float *loss, *lse_out, *total;
    unsigned int *ticket;
    // kProb
    const float *lse;          // [count]
    const float *weight;       // [count], NULL: all equal
    // kGrad, dH
    int dh_tiles_n;            // 0: not wanted
    float *slab;               // [splits][T][D rounded up], fp32 sums over the pieces so far
    int64_t slab_stride, ld_slab;
    int splits;
    int first, last;           // first piece: the slab holds nothing yet; last: dH is written (splits == 1)
    const int *rows;           // [count]: token of a packed row
    __nv_bfloat16 *dh;
    int64_t lddh;
    int dw_tiles_m;            // kGrad, dW (through tmap_out): rows of tiles, 0: not wanted
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

// 64 bf16 of row `r` of a staging tile in TMA's 128-byte swizzle: 16-byte piece j lies at j ^ (r & 7).
__device__ __forceinline__ void stage_row64(unsigned char *tile, int r, int first_piece, const float (&v)[32]) {
    unsigned char *row = tile + r * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4 *>(row + (((first_piece + q) ^ (r & 7)) << 4)) =
            make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                       pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
}

// What the tokens' slots give: lse and loss of row `row` from maximum and sum, and where they go.
__device__ __forceinline__ double finish_row(int row, float top, float sum, const float *target_logit, const int *rows, float *loss,
                                             float *lse) {
    const double l = static_cast<double>(top) * kLn2 + log(static_cast<double>(sum));
    const double x = l - static_cast<double>(__ldcg(target_logit + row));
    const int token = rows[row];
    if (lse) lse[token] = static_cast<float>(l);
    if (loss) loss[token] = static_cast<float>(x);
    return x;
}
// Joins two maxima (times log2 e) with their sums.
__device__ __forceinline__ void join(float &top, float &sum, float m, float s) {
    const float now = fmaxf(top, m);
    const float ref = now == -INFINITY ? 0.0f : now;
    sum = sum * ex2(top - ref) + s * ex2(m - ref);
    top = now;
}

template <int MODE, int TILING>
__global__ void __launch_bounds__(NUM_THREADS, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_a2, const __grid_constant__ CUtensorMap tmap_b2,
                 const __grid_constant__ CUtensorMap tmap_out, const Args a) {
    using S = Shape<MODE, TILING>;
    constexpr bool PAIR = S::PAIR;
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
        if (MODE == kGrad) {
            prefetch_tmap(&tmap_a2);
            prefetch_tmap(&tmap_b2);
        }
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

    // Work items, dealt out in turn: kLse, kProb: tiles of tokens x classes.  kGrad: (range of classes,
    // tile) of dH = G W, tokens x D, then tiles of dW = G^T H, classes x D.
    // columns per tile and per epilogue warp
    constexpr bool WIDE = TILING == kPairs || MODE == kGrad;
    const int bn = WIDE ? BN : a.bn, half_n = bn / 2;
    const int counted = a.sc->count;
    const int count_tiles = (counted + BM - 1) / BM;
    const int tiles_n = MODE == kGrad ? a.dh_tiles_n : (a.n + bn - 1) / bn;
    const int tiles = count_tiles * tiles_n;
    const int splits = MODE == kGrad ? a.splits : 1;
    const int dw_tiles_n = MODE == kGrad ? (a.n + BN - 1) / BN : 0;
    const int first_dw = tiles * splits, items = first_dw + (MODE == kGrad ? a.dw_tiles_m * dw_tiles_n : 0);
    const int k_blocks = (a.k + BK - 1) / BK, dw_k_blocks = (counted + BK - 1) / BK;
    const int kb_per = (k_blocks + splits - 1) / splits;
    struct Item {
        int tm, tn, split, kb0, nkb;
        bool dw;
    };
    // Tiles in groups of GROUP_M tile rows, column by column inside a group, so that the units running
    // at the same time share panels in L2.  An item without K blocks (no token counts, or a short last
    // piece) has an all-zero accumulator and takes no part in the barriers.
    auto item_at = [&](int i) {
        Item it;
        it.dw = MODE == kGrad && i >= first_dw;
        const int cols = it.dw ? dw_tiles_n : tiles_n, rows = it.dw ? a.dw_tiles_m : count_tiles;
        it.split = it.dw || MODE != kGrad ? 0 : i / tiles;
        const int t = it.dw ? i - first_dw : i - it.split * tiles;
        const int per_group = GROUP_M * cols;
        const int g = t / per_group;
        const int first_m = g * GROUP_M;
        const int in_group = min(GROUP_M, rows - first_m);
        const int r = t - g * per_group;
        it.tm = first_m + r % in_group;
        it.tn = r / in_group;
        it.kb0 = it.split * kb_per;
        it.nkb = it.dw ? dw_k_blocks : max(0, min(k_blocks, it.kb0 + kb_per) - it.kb0);
        return it;
    };
    // The MMA issuer and the epilogue go through the accumulators alike: the other one for each segment of kLse and
    // for each item of kProb and kGrad, but a long item (more than `segment` K blocks) and the one behind it share
    // theirs, since the other holds the long item's sum.  `phases`: a bit per accumulator, its barriers' parity.
    constexpr int segment = kSumBlocks[MODE];
    auto is_long = [](const Item &it) { return MODE != kLse && it.nkb > segment; };

    if (warp == 0) {
        // ---------------- TMA producer (every CTA) ----------------
        if (lane == 0) {
            uint32_t step = 0;
            bool ok = true;
            for (int i = unit; i < items && ok; i += n_units) {
                const Item it = item_at(i);
                const int am = it.tm * BM + rank * HALF, first_n = it.tn * bn + rank * HALF;
                for (int kb = it.kb0; kb < it.kb0 + it.nkb; ++kb, ++step) {
                    const int s = step % STAGES;
                    const uint32_t ph = (step / STAGES) & 1;
                    if (!mbar_wait(&empty[s], ph ^ 1, a.status, 401)) { ok = false; break; }
                    unsigned char *sa = smem + s * STAGE_BYTES, *sb = sa + A_BYTES;
                    // the leader's barrier collects the bytes of all loads of the pair
                    if (leader) mbar_expect_tx(&full[s], WIDE ? (PAIR ? 2 : 1) * STAGE_BYTES : A_BYTES + bn * BK * 2);
                    const uint32_t bar = PAIR ? map_to_cta(smem_u32(&full[s]), 0) : 0;
                    auto load = [&](unsigned char *dst, const CUtensorMap *map, int x, int y) {
                        if (PAIR) tma_load_2d_pair(dst, map, x, y, bar);
                        else tma_load_2d(dst, map, x, y, &full[s]);
                    };
                    if (it.dw) {              // G: 64 tokens x 128 classes, classes contiguous
                        load(sa, &tmap_a2, am, kb * BK);
                        load(sa + CHUNK_BYTES, &tmap_a2, am + 64, kb * BK);
                    } else {                  // H or G: 128 tokens x 64
                        load(sa, &tmap_a, kb * BK, am);
                    }
                    if (MODE == kGrad) {      // W or H: 64 rows x the tile's columns of D
                        const CUtensorMap *map = it.dw ? &tmap_b2 : &tmap_b;
                        const int y = (it.dw ? 0 : a.w_row0) + kb * BK;
#pragma unroll
                        for (int c = 0; c < S::B_BYTES / CHUNK_BYTES; ++c) load(sb + c * CHUNK_BYTES, map, first_n + c * 64, y);
                    } else if (WIDE) {        // W: the tile's classes x 64
                        load(sb, &tmap_b, kb * BK, a.w_row0 + first_n);
                    } else {                  // in boxes of 64 classes
                        for (int c = 0; c < bn; c += 64) load(sb + c * BK * 2, &tmap_b, kb * BK, a.w_row0 + first_n + c);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader CTA only) ----------------
        if (leader && lane == 0) {
            constexpr bool B_MN = MODE == kGrad;
            uint32_t step = 0, phases = 0;
            int buf = 0;
            bool ok = true;
            for (int i = unit; i < items && ok; i += n_units) {
                const Item it = item_at(i);
                const uint32_t idesc = it.dw ? umma_idesc_bf16(BM, BN, 1, 1) : umma_idesc_bf16(BM, bn, B_MN, 0);
                // 16 K values further: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major tile
                const uint64_t a_step = it.dw ? 2048 / 16 : 32 / 16;
                constexpr uint64_t b_step = B_MN ? 2048 / 16 : 32 / 16;
                for (int first = 0; first < it.nkb && ok; first += segment) {
                    if (!mbar_wait(&acc_empty[buf], (phases >> buf & 1) ^ 1, a.status, 402)) { ok = false; break; }
                    phases ^= 1u << buf;
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + buf * BN;
                    const int n = min(segment, it.nkb - first);
                    for (int kb = 0; kb < n; ++kb, ++step) {
                        const int s = step % STAGES;
                        const uint32_t ph = (step / STAGES) & 1;
                        if (!mbar_wait(&full[s], ph, a.status, 403)) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t sa = smem_u32(smem + s * STAGE_BYTES);
                        const uint64_t da = umma_desc_sw128(sa, it.dw ? CHUNK_BYTES : 16, 1024);
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
                    if (!is_long(it)) buf ^= 1;
                }
            }
        }
    } else {
        // ---------------- epilogue (every CTA): a thread owns a row and half of the tile's columns ----------------
        const int lane_group = warp & 3, half = (warp - 2) >> 2;
        const int r = lane_group * 32 + lane;                    // row of this CTA's part of the tile
        // results pass through a staging tile of the warp's own: no warp waits for another
        unsigned char *stage = smem + L.out.offset + (warp - 2) * S::OUT_BUFFERS * STORE_BYTES;
        uint32_t phases = 0;
        int buf = 0;
        bool ok = true;
        const float factor = MODE == kGrad ? a.sc->factor : 0.0f;
        float top = -INFINITY, sum = 0.0f;
        for (int i = unit; i < items && ok; i += n_units) {
            const Item it = item_at(i);
            const int row0 = it.tm * BM + rank * HALF, row = row0 + r;
            const int col0 = it.tn * bn + half * half_n;    // of this piece, or of D
            const bool in = row < counted;               // (dW's rows are classes: the tensor map cuts them)
            int target = -1;                             // relative to col0
            float lse2 = 0.0f, g = 0.0f;
            int token = 0;
            if (MODE != kGrad && in) target = a.target[row] - a.v0 - col0;
            if (MODE == kProb && in) {
                lse2 = static_cast<float>(static_cast<double>(a.lse[row]) * 1.4426950408889634074);
                const float largest = a.sc->largest;
                g = a.weight == nullptr ? 1.0f : largest > 0.0f ? a.weight[row] / largest : a.weight[row];
            }
            if (MODE == kGrad && !it.dw && in && a.last) token = a.rows[row];

            auto acquire = [&]() {
                if (!mbar_wait(&acc_full[buf], phases >> buf & 1, a.status, 404)) ok = false;
                phases ^= 1u << buf;
                tc_fence_after();
            };
            auto release = [&]() {   // the accumulator is free once every CTA has drained its rows
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
                    else mbar_arrive(&acc_empty[buf]);
                }
                if (!is_long(it)) buf ^= 1;
            };
            auto tmem_at = [&](int which, int column) {
                return tmem_base + (static_cast<uint32_t>(lane_group * 32) << 16) + static_cast<uint32_t>(which * BN + half * half_n + column);
            };
            auto columns = [&](int ch, float (&v)[32]) {
                uint32_t x[32];
                tmem_ld_32x32(tmem_at(buf, ch * 32), x);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(x[j]);
            };
            auto add_columns = [&](int which, int ch, float (&v)[32]) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t x[16];
                    tmem_ld_32x16(tmem_at(which, ch * 32 + q * 16), x);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[q * 16 + j] += __uint_as_float(x[j]);
                }
            };

            if constexpr (MODE == kLse) {
                float acc[4][32];
                for (int first = 0; first < it.nkb; first += segment) {
                    acquire();
                    if (!ok) break;
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        if (!WIDE && ch * 32 >= half_n) break;
                        if (first == 0) columns(ch, acc[ch]);
                        else add_columns(buf, ch, acc[ch]);
                    }
                    release();
                }
                if (!ok) break;
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    if (!WIDE && ch * 32 >= half_n) break;
                    const int col = col0 + ch * 32;
                    float (&v)[32] = acc[ch];
                    const int at = target - ch * 32;   // the target's place among these 32, if it is one of them
                    if (at >= 0 && at < 32) {
                        float x = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) x = j == at ? v[j] : x;
                        a.target_logit[row] = x;
                    }
                    if (col + 32 > a.n) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col + j >= a.n) v[j] = -INFINITY;
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
                if (!a.running) {   // one slot per tile and half
                    if (in) a.partial[(a.part0 + it.tn * 2 + half) * a.ld_partial + row] = make_float2(top, sum);
                    top = -INFINITY;
                    sum = 0.0f;
                }
            } else {
                const bool staged = MODE == kProb || it.dw;   // through shared memory; dH's rows are scattered to their tokens
                for (int first = 0; is_long(it) && first + segment < it.nkb && ok; first += segment) {   // all segments but the last
                    acquire();
                    if (!ok) break;
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        if (!WIDE && ch * 32 >= half_n) break;
                        float v[32];
                        uint32_t x[32];
                        columns(ch, v);
                        if (first) add_columns(buf ^ 1, ch, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(v[j]);
                        tmem_st_32x32(tmem_at(buf ^ 1, ch * 32), x);
                    }
                    tmem_st_wait();
                    release();
                }
                if (it.nkb && ok) acquire();
                if (!ok) break;
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {   // 64 columns
                    if (!WIDE && part * 64 >= half_n) break;
                    const int col = col0 + part * 64;
                    unsigned char *tile = stage + (S::OUT_BUFFERS == 2 ? part : 0) * STORE_BYTES;
                    if (staged) {
                        // what used this staging tile before has left it
                        if (lane == 0) tma_store_wait_read<S::OUT_BUFFERS - 1>();
                        __syncwarp();
                    }
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const int ch = part * 2 + sub, c = col + sub * 32;
                        float v[32];
                        if (it.nkb) {
                            columns(ch, v);
                            if (is_long(it)) add_columns(buf ^ 1, ch, v);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.0f;
                        }
                        if ((ch + 1) * 32 == half_n && it.nkb) release();
                        if (MODE == kProb) {
                            const int at = target - ch * 32;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                float p = ex2(fmaf(v[j], kLog2e, -lse2));
                                if (j == at) p -= 1.0f;
                                v[j] = in ? p * g : 0.0f;
                            }
                            stage_row64(tile, lane, sub * 4, v);
                        } else if (it.dw) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= factor;
                            stage_row64(tile, lane, sub * 4, v);
                        } else if (in && c < a.n) {
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
                                store_row32(a.dh + static_cast<int64_t>(token) * a.lddh + c, v, a.n - c);
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    *reinterpret_cast<float4 *>(s + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                            }
                        }
                    }
                    const int first_row = row0 + lane_group * 32;
                    if (staged) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            // rows behind the matrix and columns behind its last are cut off by the tensor map
                            if (col < a.n && (MODE == kProb || first_row < a.k)) tma_store_2d(&tmap_out, tile, col, first_row);
                            tma_store_commit();
                        }
                    }
                }
            }
        }
        if (S::STORE && lane == 0) tma_store_wait_all<0>();
        if (MODE == kLse && a.running) {
            // one slot per unit: the halves of the columns join in shared memory
            float2 *halves = reinterpret_cast<float2 *>(smem + L.out.offset);
            if (half == 1) halves[r] = make_float2(top, sum);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (half == 0) {
                const float2 o = halves[r];
                join(top, sum, o.x, o.y);
                const int row = rank * HALF + r;
                if (row < counted) a.partial[row * a.ld_partial + a.part0 + unit] = make_float2(top, sum);
            }
            __threadfence();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();   // no CTA may leave while its partner can still signal into it
    if (warp == 1) {
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
    if constexpr (MODE == kLse) {
        if (!a.running || !a.finish) return;
        // The last CTA to come here joins the units' slots: a warp per row, lanes across the slots.
        __shared__ bool last_block;
        __shared__ double sums[NUM_THREADS / 32];
        if (threadIdx.x == 0) last_block = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
        __syncthreads();
        if (!last_block) return;
        __threadfence();
        const int slots = a.part0 + n_units;
        double mine = 0.0;
        for (int row = warp; row < counted; row += NUM_THREADS / 32) {
            float m = -INFINITY, t = 0.0f;
            for (int p = lane; p < slots; p += 32) {
                const float2 v = __ldcg(a.partial + row * a.ld_partial + p);
                join(m, t, v.x, v.y);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, o), t2 = __shfl_xor_sync(0xffffffffu, t, o);
                // the same order of the two on both sides, so that all lanes hold the same bits
                float hi_m = lane & o ? m2 : m, hi_t = lane & o ? t2 : t;
                join(hi_m, hi_t, lane & o ? m : m2, lane & o ? t : t2);
                m = hi_m;
                t = hi_t;
            }
            if (lane == 0) mine += finish_row(row, m, t, a.target_logit, a.rows, a.loss, a.lse_out);
        }
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {
            double all = 0.0;
            for (int w = 0; w < NUM_THREADS / 32; ++w) all += sums[w];
            if (a.total) {
                a.total[0] = a.sc->bad ? __int_as_float(0x7fffffff) : static_cast<float>(all);
                a.total[1] = static_cast<float>(counted);
            }
            *a.ticket = 0;
        }
    }
}

// What the kernels that pick out the counted tokens read and write.
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
    // packing
    const __nv_bfloat16 *H;
    int64_t ldh;
    int D;
    __nv_bfloat16 *Hc;
    int64_t ldc;
    __nv_bfloat16 *dH;           // backward: zeroed where a token does not count
    int64_t lddh;

    __device__ bool keeps(int64_t t) const { return t != ignore && t >= 0 && t < V; }
    __device__ void skip(int64_t i, int64_t t) const {   // results of a token that does not count
        const float v = t != ignore ? __int_as_float(0x7fffffff) : 0.0f;
        if (loss_out) loss_out[i] = v;
        if (lse_out) lse_out[i] = v;
    }
    __device__ void keep(int at, int64_t i, int64_t t) const {
        rows[at] = (int)i;
        target[at] = (int)t;
        if (lse) lse_c[at] = lse[i];
        if (dloss) weight_c[at] = dloss[i];
    }
    __device__ void scalars(int count, int bad, float largest) const {
        Scalars s;
        s.count = count;
        s.bad = bad;
        // No weight but 0 (or none that is finite): G takes them as they are.  The same where the largest is so large
        // that ordinary ones over it, or the factor itself, could leave fp32's range.
        constexpr float kHuge = 1.1529215e18f;     // 2^60
        s.largest = largest <= kHuge && fabsf(scale) <= kHuge ? largest : 0.0f;
        s.factor = count == 0 ? 0.0f : dloss ? (s.largest > 0.0f ? scale * s.largest : scale) : total ? scale / total[1] : 0.0f;
        *sc = s;
    }
};

// 8 elements that may lie on any 2-byte boundary, without a read outside them.
__device__ __forceinline__ uint4 load8(const __nv_bfloat16 *p) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) return __ldcs(reinterpret_cast<const uint4 *>(p));
    if ((reinterpret_cast<uintptr_t>(p) & 3) == 0) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
        return make_uint4(q[0], q[1], q[2], q[3]);
    }
    const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
    const uint32_t *q = reinterpret_cast<const uint32_t *>(h + 1);
    const uint32_t first = h[0], w0 = q[0], w1 = q[1], w2 = q[2], last = h[7];
    return make_uint4(first | w0 << 16, __funnelshift_l(w0, w1, 16), __funnelshift_l(w1, w2, 16), w2 >> 16 | last << 16);
}
__device__ __forceinline__ void copy8(const __nv_bfloat16 *src, __nv_bfloat16 *dst, int n) {
    if (n >= 8) *reinterpret_cast<uint4 *>(dst) = load8(src);
    else
        for (int j = 0; j < n; ++j) dst[j] = src[j];
}

// A block's part of packing: the row of the token `from` (< 0: a row of zeros) becomes packed row `r`.
__device__ __forceinline__ void pack_row(const PrepareArgs &a, int r, int from) {
    __nv_bfloat16 *dst = a.Hc + r * a.ldc;
    if (from >= 0) {
        const __nv_bfloat16 *src = a.H + from * a.ldh;
        for (int j = threadIdx.x * 8; j < a.D; j += blockDim.x * 8) copy8(src + j, dst + j, a.D - j);
    } else {
        for (int j = threadIdx.x * 8; j < a.ldc; j += blockDim.x * 8) *reinterpret_cast<uint4 *>(dst + j) = make_uint4(0, 0, 0, 0);
    }
}
__device__ __forceinline__ void zero_gradient_row(const PrepareArgs &a, int64_t token) {
    for (int j = threadIdx.x; j < a.D; j += blockDim.x) a.dH[token * a.lddh + j] = __float2bfloat16_rn(0.0f);
}

// Where the counted tokens' rows go: a block per token finds its place among the counted ones from the counts
// of the segments before its own and the targets of its own segment.  Up to kSmallT tokens are one segment
// and one launch; longer lists have segments of 256 whose counts a first launch leaves (one block that listed
// all tokens took 11 us for 6007 of them).
constexpr int kSmallT = 1024, kSegment = 256;
struct SegmentCount {
    int count, bad;
    float top;
};

// Kept and bad tokens and the largest weight among up to 8 tokens per thread of a block of 128; every
// thread gets the block's totals, `before` the number kept in front of the thread's first.
struct Tally {
    int before, count, bad;
    float top;
};
template <int PER>
__device__ __forceinline__ Tally tally(const PrepareArgs &a, int64_t first, const int64_t (&t)[PER]) {
    __shared__ int counts[4], bads[4];
    __shared__ float tops[4];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    int mine = 0, bad = 0;
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool keep = a.keeps(t[k]);
        mine += keep;
        bad += !keep && t[k] != a.ignore;
        if (keep && a.dloss) {
            const float g = fabsf(a.dloss[first + k]);
            if (g < INFINITY) top = fmaxf(top, g);    // an infinite or NaN weight is its own token's affair
        }
    }
    Tally r;
    r.before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, r.before, o);
        if (lane >= o) r.before += up;
    }
    top = warp_max(top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bad += __shfl_xor_sync(0xffffffffu, bad, o);
    if (lane == 31) {
        counts[wid] = r.before;
        bads[wid] = bad;
        tops[wid] = top;
    }
    r.before -= mine;
    __syncthreads();
    r.count = 0;
    r.bad = 0;
    r.top = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wid) r.before += counts[w];
        r.count += counts[w];
        r.bad += bads[w];
        r.top = fmaxf(r.top, tops[w]);
    }
    return r;
}
template <int PER>
__device__ __forceinline__ void load_targets(const PrepareArgs &a, int64_t first, int64_t end, int64_t (&t)[PER]) {
#pragma unroll
    for (int k = 0; k < PER; ++k) t[k] = first + k < end ? a.targets[first + k] : a.ignore;
}

__global__ void __launch_bounds__(128) xent_count_kernel(const PrepareArgs a, SegmentCount *segments) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kSegment + threadIdx.x * 2;
    int64_t t[2];
    load_targets(a, first, a.T, t);
    const Tally r = tally(a, first, t);
    if (threadIdx.x == 0) segments[blockIdx.x] = {r.count, r.bad, r.top};
}

// Block i: packs token i's row if it counts; writes zeros as packed row i if that lies behind the last
// counted one and before a multiple of 64 (such rows are K rows of dW's product).
template <int PER>
__global__ void __launch_bounds__(128) xent_gather_kernel(const PrepareArgs a, const SegmentCount *segments, int n_segments) {
    __shared__ int place, sums[3][4];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, i = blockIdx.x;
    const int segment = PER * 128 < kSmallT ? i / kSegment : 0;
    const int64_t base = static_cast<int64_t>(segment) * (PER * 128), first = base + threadIdx.x * PER;
    int64_t t[PER];
    load_targets(a, first, min(base + PER * 128, static_cast<int64_t>(a.T)), t);
    const Tally own = tally(a, first, t);
    int count = own.count, bad = own.bad, earlier = 0;
    float top = own.top;
    if (PER * 128 < kSmallT) {      // the other segments' counts
        int all = 0;
        bad = 0;
        top = 0.0f;
        for (int s = threadIdx.x; s < n_segments; s += 128) {
            const SegmentCount c = segments[s];
            all += c.count;
            if (s < segment) earlier += c.count;
            bad += c.bad;
            top = fmaxf(top, c.top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            all += __shfl_xor_sync(0xffffffffu, all, o);
            earlier += __shfl_xor_sync(0xffffffffu, earlier, o);
            bad += __shfl_xor_sync(0xffffffffu, bad, o);
        }
        top = warp_max(top);
        __shared__ float tops[4];
        if (lane == 0) {
            sums[0][wid] = all;
            sums[1][wid] = earlier;
            sums[2][wid] = bad;
            tops[wid] = top;
        }
        __syncthreads();
        count = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
        earlier = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
        bad = sums[2][0] + sums[2][1] + sums[2][2] + sums[2][3];
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    }
    if (i >= count && i < (count + BK - 1) / BK * BK) pack_row(a, i, -1);
    if (i == 0 && threadIdx.x == 0) a.scalars(count, bad, top);
    if (i >= a.T) return;
    // the thread that holds token i's target knows its place
    int at = earlier + own.before;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool keep = a.keeps(t[k]);
        if (first + k == i) {
            place = keep ? at : -1;
            if (keep) a.keep(at, i, t[k]);
            else a.skip(i, t[k]);
        }
        at += keep;
    }
    __syncthreads();
    if (place >= 0) pack_row(a, place, i);
    else if (a.dH) zero_gradient_row(a, i);
}

// Rows of W whose pitch or address TMA cannot take, packed to a pitch of 16 bytes' multiple.
__global__ void __launch_bounds__(256)
xent_pack_weight_kernel(const __nv_bfloat16 *W, int64_t ldw, int rows, int D, __nv_bfloat16 *Wc, int64_t ldc) {
    pdl_launch_dependents();
    pdl_wait();
    const int groups = static_cast<int>(ldc / 8);    // 8 elements each
    const int64_t all = static_cast<int64_t>(rows) * groups;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / groups;
        const int j = static_cast<int>(i - row * groups) * 8;
        copy8(W + row * ldw + j, Wc + row * ldc + j, D - j);
    }
}

// The same way back: packed rows of dW to rows on any address.  A warp writes a row as consecutive words.
__global__ void __launch_bounds__(256)
xent_unpack_kernel(const __nv_bfloat16 *packed, int64_t ldp, int rows, int D, __nv_bfloat16 *dW, int64_t lddw) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += static_cast<int64_t>(gridDim.x) * 8) {
        const uint32_t *src = reinterpret_cast<const uint32_t *>(packed + row * ldp);    // 16-byte aligned, padded to 8 elements
        unsigned short *dst = reinterpret_cast<unsigned short *>(dW + row * lddw);
        const int first = (reinterpret_cast<uintptr_t>(dst) & 2) ? 1 : 0;    // elements before the first whole word
        const int words = (D - first) / 2;
        uint32_t *out = reinterpret_cast<uint32_t *>(dst + first);
        if (lane == 0 && first) dst[0] = static_cast<unsigned short>(src[0]);
        if (lane == 1 && first + 2 * words < D) dst[D - 1] = static_cast<unsigned short>(src[(D - 1) / 2] >> ((D - 1) % 2 * 16));
        for (int k0 = 0; k0 < words; k0 += 128) {        // four words a lane in flight
            uint32_t w[4], edge[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = k0 + q * 32 + lane;
                w[q] = k < words + first ? src[k] : 0;
                edge[q] = first && lane == 31 && k < words ? src[k + 1] : 0;     // (2 (k + 1) <= D - 1: inside the padded row)
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = k0 + q * 32 + lane;
                uint32_t next = __shfl_down_sync(0xffffffffu, w[q], 1);
                if (lane == 31) next = edge[q];
                if (k < words) out[k] = first ? w[q] >> 16 | next << 16 : w[q];
            }
        }
    }
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
    if (row < count) {
        for (int p = deep; p < parts; p += 8 * 32) {   // eight slots at a time: their loads and exponentials overlap
            float2 v[8];
            float m = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = p + k * 32 < parts ? __ldcs(partial + (p + k * 32) * ld_partial + row) : make_float2(-INFINITY, 0.0f);
                m = fmaxf(m, v[k].x);
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            float s = sum * ex2(top - ref);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k].y * ex2(v[k].x - ref);
            sum = s;
            top = m;
        }
    }
    tops[deep][lane] = top;
    sums[deep][lane] = sum;
    __syncthreads();
    if (deep == 0) {
        double mine = 0.0;
        if (row < count) {
            top = -INFINITY;
#pragma unroll
            for (int d = 0; d < 32; ++d) top = fmaxf(top, tops[d][lane]);
            const float ref = top == -INFINITY ? 0.0f : top;
            sum = 0.0f;
#pragma unroll
            for (int d = 0; d < 32; ++d) sum += sums[d][lane] * ex2(tops[d][lane] - ref);
            mine = finish_row(row, top, sum, target_logit, rows, loss, lse);
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

// dH of split sums: four columns a thread, `depth` threads (1 to 8) for the ranges of a row, 8 / depth rows a block.
__global__ void __launch_bounds__(256)
xent_dh_finish_kernel(const float *slab, int64_t slab_stride, int64_t ld_slab, int splits, int depth, const int *rows,
                      const Scalars *sc, int D, __nv_bfloat16 *dH, int64_t lddh) {
    __shared__ float4 part[8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, deep = wid % depth;
    const int row = blockIdx.x * (8 / depth) + wid / depth;
    const int j = (blockIdx.y * 32 + lane) * 4;
    const bool in = row < sc->count && j < D;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (in) {
        const float *src = slab + row * ld_slab + j;     // rows of the slab are padded to 32 columns
#pragma unroll 8
        for (int k = deep; k < splits; k += depth) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + k * slab_stride));
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
    }
    part[wid][lane] = s;
    __syncthreads();
    if (deep != 0 || !in) return;
    for (int k = 1; k < depth; ++k) {
        const float4 v = part[wid + k][lane];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    const float factor = sc->factor;
    __nv_bfloat16 *dst = dH + rows[row] * lddh + j;
    if (j + 4 <= D && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16(s.x * factor, s.y * factor), pack_bf16(s.z * factor, s.w * factor));
    } else {
        const float v[4] = {s.x, s.y, s.z, s.w};
        for (int k = 0; k < 4 && j + k < D; ++k) dst[k] = __float2bfloat16_rn(v[k] * factor);
    }
}

// ---- host side -----------------------------------------------------------------------------------

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int segment_count(int64_t T) { return (int)((T + kSegment - 1) / kSegment); }

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
    Tiling tiling;

    bool pack_w() const { return (reinterpret_cast<uintptr_t>(W) & 15) != 0 || ldw % 8 != 0; }
    int64_t dp() const { return up(D, 8); }
    int tiles(int64_t n) const { return (int)((n + 255) / 256); }
};

int map_of(gb200_ctx *ctx, const void *p, int64_t cols, int64_t rows, int64_t ld, int box_rows, CUtensorMap *out) {
    return get_tmap_2d(ctx, p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)cols, (uint64_t)rows, (uint64_t)ld * 2, 64,
                       (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B, out);
}

// Rows of tiles cost what they hold, used or not; a single CTA's 128 rows cost more than half a pair's 256,
// whose B tiles two CTAs share.  Measured over 65536 x 2048, singles / pairs: 300 tokens 96 / 98 us, 600
// tokens 143 / 153 us (but the gradients' step 196 / 195), 1100 tokens 246 / 233 us.
Tiling tiling(int T) {
    if (T <= kFewT) return kFew;
    const int pairs = (T + 255) / 256 * 256, singles = (T + 127) / 128 * 128;
    return singles * 5 < pairs * 4 ? kSingles : kPairs;
}
int units(const Call &c) { return std::max(c.tiling == kPairs ? c.ctx->sm_count / 2 : c.ctx->sm_count, 1); }
int64_t tile_rows(const Call &c, int64_t rows) {
    const int bm = c.tiling == kPairs ? 256 : 128;
    return (rows + bm - 1) / bm;
}
int w_box(const Call &c) { return c.tiling == kPairs ? HALF : 64; }   // rows of W per load
int a_rows(const Call &c) { return c.tiling == kFew ? kFewT : HALF; }
// The vocabulary in equal pieces of at most `most` classes (a multiple of 256).
int64_t equal_pieces(int64_t V, int64_t most) {
    if (V <= most) return V;
    const int64_t n = (V + most - 1) / most;
    return up((V + n - 1) / n, 256);
}

// Columns per tile on single CTAs: rounds of tiles over the SMs times a tile's width, each tile charged 32
// columns for what it costs besides.  21 x 9728 x 1344: 76 tiles of 128 instead of 38 of 256.
int pick_columns(const Call &c, int64_t rows, int64_t n, int least) {
    if (c.tiling == kPairs) return BN;
    int best = BN;
    int64_t best_cost = INT64_MAX;
    for (int w = BN; w >= least; w /= 2) {
        const int64_t cost = (rows * ((n + w - 1) / w) + units(c) - 1) / units(c) * (w + 32);
        if (cost < best_cost) {
            best_cost = cost;
            best = w;
        }
    }
    return best;
}

struct Maps {
    CUtensorMap a, b, a2, b2, out;
};

template <int MODE, int TILING>
int launch_as(const Call &c, const Maps &m, int64_t n_units, const Args &a) {
    using S = Shape<MODE, TILING>;
    constexpr int bytes = S::layout.dynamic_bytes;
    auto kern = xent_gemm_kernel<MODE, TILING>;
    const int rc = ensure_dynamic_smem(c.ctx, kern, bytes);
    if (rc) return rc;
    GB200_CUDA_TRY(launch_pdl_cluster(kern, dim3((unsigned)(n_units * (S::PAIR ? 2 : 1))), dim3(NUM_THREADS), (size_t)bytes,
                                      c.stream, S::PAIR ? 2u : 1u, m.a, m.b, m.a2, m.b2, m.out, a));
    static const char *const names[] = {"xent_gemm_kernel<lse>", "xent_gemm_kernel<prob>", "xent_gemm_kernel<grad>"};
    return after_launch(c.ctx, names[MODE]);
}

// Returns the number of units launched (CTAs or pairs) through *used.
template <int MODE>
int launch(const Call &c, const Maps &m, int64_t items, Args a, int *used = nullptr) {
    const int64_t n = std::min<int64_t>(units(c), items);
    if (used) *used = (int)n;
    a.status = c.ctx->d_status;
    if (c.tiling == kPairs) return launch_as<MODE, kPairs>(c, m, n, a);
    if constexpr (MODE != kGrad)    // (G has 128 rows whatever the tokens' number)
        if (c.tiling == kFew) return launch_as<MODE, kFew>(c, m, n, a);
    return launch_as<MODE, kSingles>(c, m, n, a);
}

int gather(const Call &c, const PrepareArgs &p, SegmentCount *segments) {
    const dim3 blocks((unsigned)up(c.T, BK));
    if (c.T <= kSmallT) {
        GB200_CUDA_TRY(launch_pdl(xent_gather_kernel<kSmallT / 128>, blocks, dim3(128), 0, c.stream, p, segments, 1));
        return after_launch(c.ctx, "xent_gather_kernel");
    }
    const int n = segment_count(c.T);
    GB200_CUDA_TRY(launch_pdl(xent_count_kernel, dim3((unsigned)n), dim3(128), 0, c.stream, p, segments));
    const int rc = after_launch(c.ctx, "xent_count_kernel");
    if (rc) return rc;
    GB200_CUDA_TRY(launch_pdl(xent_gather_kernel<kSegment / 128>, blocks, dim3(128), 0, c.stream, p, segments, n));
    return after_launch(c.ctx, "xent_gather_kernel");
}

int pack_weight(const Call &c, int64_t v0, int64_t rows, __nv_bfloat16 *Wc) {
    const int64_t groups = rows * (c.dp() / 8);
    const int64_t blocks = std::min<int64_t>((groups + 1023) / 1024, (int64_t)c.ctx->sm_count * 32);
    GB200_CUDA_TRY(launch_pdl(xent_pack_weight_kernel, dim3((unsigned)blocks), dim3(256), 0, c.stream, c.W + v0 * c.ldw, c.ldw,
                              (int)rows, c.D, Wc, c.dp()));
    return after_launch(c.ctx, "xent_pack_weight_kernel");
}

int unpack_gradient(const Call &c, const __nv_bfloat16 *packed, int64_t rows, __nv_bfloat16 *dW, int64_t lddw) {
    const int64_t blocks = std::min<int64_t>((rows + 7) / 8, (int64_t)c.ctx->sm_count * 64);
    GB200_CUDA_TRY(launch_pdl(xent_unpack_kernel, dim3((unsigned)blocks), dim3(256), 0, c.stream, packed, c.dp(), (int)rows, c.D, dW,
                              lddw));
    return after_launch(c.ctx, "xent_unpack_kernel");
}

PrepareArgs prepare_args(const Call &c, Scalars *sc, int *rows, int *target, __nv_bfloat16 *Hc) {
    PrepareArgs p{};
    p.targets = c.targets;
    p.T = c.T;
    p.V = c.V;
    p.ignore = c.ignore;
    p.rows = rows;
    p.target = target;
    p.sc = sc;
    p.H = c.H;
    p.ldh = c.ldh;
    p.D = c.D;
    p.Hc = Hc;
    p.ldc = c.dp();
    return p;
}

int forward(const Call &c, float *loss, float *lse, float *total) {
    // the whole vocabulary at once, unless W has to be packed first
    const int64_t piece = c.pack_w() ? equal_pieces(c.V, std::max<int64_t>(kPieceBytes / (c.dp() * 2) / 256 * 256, 256)) : c.V;
    // one row of tiles: a slot per unit and piece, else two per tile column
    const bool running = tile_rows(c, c.T) == 1;
    const int64_t pieces = (c.V + piece - 1) / piece;
    const int bn = pick_columns(c, tile_rows(c, c.T), piece, 64);
    const int64_t parts = running ? units(c) * pieces : 2 * ((c.V + bn - 1) / bn + pieces);
    Scratch s;
    int *rows, *target;
    Scalars *sc;
    SegmentCount *segments;
    float *target_logit;
    float2 *partial;
    double *block_sums;
    __nv_bfloat16 *Hc, *Wc;
    for (int pass = 0; pass < 2; ++pass) {
        s.used = 0;
        sc = s.take<Scalars>(1);
        segments = s.take<SegmentCount>(segment_count(c.T));
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
    PrepareArgs p = prepare_args(c, sc, rows, target, Hc);
    p.loss_out = loss;
    p.lse_out = lse;
    int rc = gather(c, p, segments);
    if (rc) return rc;
    Maps m;
    rc = map_of(c.ctx, Hc, c.D, c.T, c.dp(), a_rows(c), &m.a);
    if (rc) return rc;
    Args a{};
    a.sc = sc;
    a.bn = bn;
    a.k = c.D;
    a.target = target;
    a.rows = rows;
    a.partial = partial;
    a.ld_partial = running ? parts : c.T;
    a.running = running;
    a.target_logit = target_logit;
    a.loss = loss;
    a.lse_out = lse;
    a.total = total;
    a.ticket = c.ctx->tickets + kTicketXent;
    for (int64_t v0 = 0; v0 < c.V; v0 += piece) {
        const int64_t n = std::min<int64_t>(piece, c.V - v0);
        if (c.pack_w()) {
            rc = pack_weight(c, v0, n, Wc);
            if (rc) return rc;
        }
        rc = c.pack_w() ? map_of(c.ctx, Wc, c.D, n, c.dp(), w_box(c), &m.b) : map_of(c.ctx, c.W, c.D, c.V, c.ldw, w_box(c), &m.b);
        if (rc) return rc;
        m.a2 = m.b2 = m.out = m.b;
        a.n = (int)n;
        a.w_row0 = c.pack_w() ? 0 : (int)v0;
        a.v0 = (int)v0;
        a.finish = v0 + n == c.V;
        int used = 0;
        const int64_t tiles_n = (n + bn - 1) / bn;
        rc = launch<kLse>(c, m, tile_rows(c, c.T) * tiles_n, a, &used);
        if (rc) return rc;
        a.part0 += running ? used : (int)(2 * tiles_n);
    }
    if (running) return GB200_OK;
    GB200_CUDA_TRY(launch_pdl(xent_finish_kernel, dim3((unsigned)((c.T + 31) / 32)), dim3(1024), 0, c.stream, partial, (int64_t)c.T,
                              a.part0, target_logit, rows, sc, loss, lse, total, block_sums, c.ctx->tickets + kTicketXent));
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
    // (G has rows for whole tiles of tokens)
    int64_t piece = std::max<int64_t>(kPieceBytes / (2 * up(c.T, 256)) / 256 * 256, kPieceClasses);
    // dW whose rows TMA cannot write is made packed, piece by piece.  (A TMA store cuts a row off at whole 16-byte
    // pieces only: with D no multiple of 8 it would write into the gap between the rows.)
    const bool unpack = dW && ((reinterpret_cast<uintptr_t>(dW) & 15) != 0 || lddw % 8 != 0 || c.D % 8 != 0);
    if (c.pack_w() || unpack) piece = std::min(piece, std::max<int64_t>(kPieceBytes / (c.dp() * 2) / 256 * 256, 256));
    piece = equal_pieces(c.V, piece);
    const int64_t ld_slab = up(c.D, 32), slab_stride = ld_slab * c.T, ldg = up(piece, 64);
    // The gradients' products: most of their tiles are dW's, whose rows are classes, so pairs pay from fewer tokens on
    // (290 x 87296 x 2112 534 / 550 us on pairs / single CTAs, 120 x 32768 x 1024 117 / 102 us).
    Call gc = c;
    gc.tiling = c.T > 128 ? kPairs : kSingles;
    const int64_t dh_tiles = tile_rows(gc, c.T) * c.tiles(c.D);
    const int splits = pick_splits(dh_tiles, up(piece, BK) / BK, units(gc), slab_stride * 4);
    const bool slab_wanted = dH && (splits > 1 || piece < c.V);
    Scratch s;
    int *rows, *target;
    Scalars *sc;
    SegmentCount *segments;
    float *lse_c, *weight_c, *slab;
    __nv_bfloat16 *Hc, *Wc, *Dc, *G;
    for (int pass = 0; pass < 2; ++pass) {
        s.used = 0;
        sc = s.take<Scalars>(1);
        segments = s.take<SegmentCount>(segment_count(c.T));
        rows = s.take<int>(c.T);
        target = s.take<int>(c.T);
        lse_c = s.take<float>(c.T);
        weight_c = s.take<float>(c.T);
        Hc = s.take<__nv_bfloat16>(up(c.T, BK) * c.dp());
        Wc = c.pack_w() ? s.take<__nv_bfloat16>(piece * c.dp()) : nullptr;
        Dc = unpack ? s.take<__nv_bfloat16>(piece * c.dp()) : nullptr;
        G = s.take<__nv_bfloat16>(up(c.T, 256) * ldg);
        slab = slab_wanted ? s.take<float>(splits * slab_stride) : nullptr;
        if (pass == 0) {
            void *base = nullptr;
            const int rc = scratch_reserve(c.ctx, s.used, c.stream, &base);
            if (rc) return rc;
            s.base = static_cast<unsigned char *>(base);
        }
    }
    PrepareArgs p = prepare_args(c, sc, rows, target, Hc);
    p.lse = lse;
    p.dloss = dloss;
    p.total = total;
    p.scale = scale;
    p.lse_c = lse_c;
    p.weight_c = weight_c;
    p.dH = dH;
    p.lddh = lddh;
    int rc = gather(c, p, segments);
    if (rc) return rc;
    Maps prob, grad;
    rc = map_of(c.ctx, Hc, c.D, up(c.T, BK), c.dp(), a_rows(c), &prob.a);
    if (!rc) rc = map_of(c.ctx, Hc, c.D, up(c.T, BK), c.dp(), BK, &grad.b2);
    if (rc) return rc;
    Args a{};
    a.sc = sc;
    a.target = target;
    a.rows = rows;
    a.lse = lse_c;
    a.weight = dloss ? weight_c : nullptr;
    a.splits = splits;
    a.slab = slab;
    a.slab_stride = slab_stride;
    a.ld_slab = ld_slab;
    a.dh = dH;
    a.lddh = lddh;
    for (int64_t v0 = 0; v0 < c.V; v0 += piece) {
        const int64_t n = std::min<int64_t>(piece, c.V - v0);
        if (c.pack_w()) {
            rc = pack_weight(c, v0, n, Wc);
            if (rc) return rc;
        }
        const void *wp = c.pack_w() ? static_cast<const void *>(Wc) : c.W;
        const int64_t w_rows = c.pack_w() ? n : c.V, w_ld = c.pack_w() ? c.dp() : c.ldw;
        rc = map_of(c.ctx, wp, c.D, w_rows, w_ld, w_box(c), &prob.b);
        if (!rc) rc = map_of(c.ctx, wp, c.D, w_rows, w_ld, BK, &grad.b);
        if (!rc) rc = map_of(c.ctx, G, n, up(c.T, 256), ldg, HALF, &grad.a);
        if (!rc) rc = map_of(c.ctx, G, n, up(c.T, 256), ldg, BK, &grad.a2);
        if (!rc) rc = map_of(c.ctx, G, n, up(c.T, 256), ldg, 32, &prob.out);
        grad.out = prob.out;
        if (!rc && dW) rc = unpack ? map_of(c.ctx, Dc, c.D, n, c.dp(), 32, &grad.out) : map_of(c.ctx, dW + v0 * lddw, c.D, n, lddw, 32, &grad.out);
        if (rc) return rc;
        prob.a2 = prob.a;
        prob.b2 = prob.b;
        a.w_row0 = c.pack_w() ? 0 : (int)v0;
        a.v0 = (int)v0;
        a.n = (int)n;
        a.k = c.D;
        a.bn = pick_columns(c, tile_rows(c, c.T), n, 128);
        rc = launch<kProb>(c, prob, tile_rows(c, c.T) * ((n + a.bn - 1) / a.bn), a);
        if (rc) return rc;
        a.n = c.D;
        a.k = (int)n;
        a.first = v0 == 0;
        a.last = v0 + n == c.V && splits == 1;
        a.dh_tiles_n = dH ? c.tiles(c.D) : 0;
        a.dw_tiles_m = dW ? (int)tile_rows(gc, n) : 0;
        rc = launch<kGrad>(gc, grad, (dH ? dh_tiles * splits : 0) + (int64_t)a.dw_tiles_m * c.tiles(c.D), a);
        if (!rc && unpack) rc = unpack_gradient(c, Dc, n, dW + v0 * lddw, lddw);
        if (rc) return rc;
    }
    if (dH && splits > 1) {
        const int depth = splits >= 32 ? 8 : splits >= 16 ? 4 : splits >= 8 ? 2 : 1, rows_per = 8 / depth;
        GB200_CUDA_TRY(launch_pdl(xent_dh_finish_kernel, dim3((unsigned)((c.T + rows_per - 1) / rows_per), (unsigned)((c.D + 127) / 128)),
                                  dim3(256), 0, c.stream, slab, slab_stride, ld_slab, splits, depth, rows, sc, c.D, dH, lddh));
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

// The loss's product on CTA pairs, as gb200_kernel_resources_query reports it.
gb200_kernel_resources linear_xent_resources() {
    return {kernel_registers(xent_gemm_kernel<kLse, kPairs>), NUM_THREADS, Shape<kLse, kPairs>::layout.dynamic_bytes, 2, 512};
}

}  // namespace gb200

using namespace gb200;

extern "C" {

int gb200_linear_xent_bf16(gb200_ctx *ctx, const void *H, int64_t ldh, const void *W, int64_t ldw, const int64_t *targets,
                           int64_t T, int64_t V, int64_t D, int64_t ignore_index, float *loss, float *lse, float *total,
                           void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check(H, ldh, W, ldw, targets, T, V, D);
    if (rc) return rc;
    // (operands of no tokens are empty and may have no address)
    GB200_REQUIRE(T == 0 || loss || lse || total, GB200_ERR_INVALID_ARG, "nothing to produce: loss, lse and total are NULL");
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
                 (int)V, (int)D, ignore_index, st, tiling((int)T)};
    return forward(c, loss, lse, total);
}

int gb200_linear_xent_bf16_backward(gb200_ctx *ctx, const void *H, int64_t ldh, const void *W, int64_t ldw,
                                    const int64_t *targets, const float *lse, const float *dloss, const float *total,
                                    int64_t T, int64_t V, int64_t D, int64_t ignore_index, float scale, void *dH,
                                    int64_t lddh, void *dW, int64_t lddw, void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check(H, ldh, W, ldw, targets, T, V, D);
    if (rc) return rc;
    GB200_REQUIRE(T == 0 || dH || dW, GB200_ERR_INVALID_ARG, "nothing to produce: dH and dW are NULL");
    GB200_REQUIRE((T == 0 && !dloss) || (dloss != nullptr) != (total != nullptr), GB200_ERR_INVALID_ARG,
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
                 (int)V, (int)D, ignore_index, st, tiling((int)T)};
    return backward(c, lse, dloss, total, scale, static_cast<__nv_bfloat16 *>(dH), lddh, static_cast<__nv_bfloat16 *>(dW), lddw);
}

}  // extern "C"
