// Softmax cross entropy over a vocabulary matrix W [V, R] (stored, or noise regenerated from a seed), loss and gradients, without
// keeping the logits l = x W^T.
//
// Everything is taken relative to the logit of the row's own target t, which a small kernel computes first:
//
//   e_v = exp(l_v - l_t),  s = sum over v != t of e_v        loss = log(1 + s)            lse = l_t + loss
//   d loss / dx = (sum over v != t of e_v w_v  -  s w_t) / (1 + s)
//
// so no running maximum is needed: the sum never falls below the target's own 1, and small losses and the gradients of tokens
// the model already knows come out of log1p and of a sum without the target, not of a difference of nearly equal numbers.  Float32
// holds e_v up to 69 above the target's logit (s below 2^100 leaves room for the gradient).  Where the row's length says that the
// largest of V random logits will lie 40 or more above the target's (|x| |w_t| / sqrt(R) is their standard deviation, largest_of(V)
// of those the mean of the largest), or over a stored matrix, whose logits need be neither independent nor about 0, where a few sampled
// ones say so (sampled_top), that estimate takes the target's place:  e_v = exp(l_v - l_t - d),  loss = log(1 + s exp(d)).  A row that
// leaves the range all the same, at either end, or whose target then turns out to be likelier than all others together, is noticed
// and done again with its true maximum (ce_far_rows).
//
// Rows whose target is ignored are left out: the remaining rows are gathered to the front, and every later kernel works on that
// many rows, a number that only the device knows.
//
//   gradient of x only (noise matrix): one pass over the vocabulary in pieces, E = exp(..) of a piece in bf16, O += E W_piece in
//       float32; the gradient is finished from O, s and the target's row.  Two products per (row, vocabulary, R).
//   stored matrix: the forward needs only s (one product); the backward recomputes each piece's logits with the final lse,
//       P = w (softmax - onehot), and takes dx += P W_piece and dW_piece = P^T x.  Four products in all.
//
// float32 operands are split into three bf16 parts each (3 x 8 = 24 significant bits) and multiplied as the six products of
// parts whose orders add up to at most two, accumulated in the same float32 accumulator: exact products, terms below 2^-24
// left out.
//
// The products run on CTA pairs (cta_group::2).  bf16: 512 x 256 tiles, two 256 x 256 accumulators that fill TMEM and take MMAs in
// turn, four 48 KB stages of TMA-fed operands; an epilogue warp takes its 32 rows x 128 columns of an accumulator into registers,
// hands the accumulator back and computes from the registers, and the MMA thread runs ahead on the first accumulator while the
// second is still being read.  (256 x 256 tiles, whose MMAs all go to one accumulator, kept the tensor pipe 62 % busy.)  Few rows
// (ce_tile_rows): 256 x 256 tiles, six 32 KB stages.  float32: the same, and the accumulators, whose additions cut instead of rounding (about
// 2^-26 of the sum per 16 products, all in one direction), are added up in the epilogue's registers every eight k-blocks.
#include <atomic>
#include <cmath>

#include "umma.cuh"
#include "umma_pipe.cuh"

namespace rdb {

using namespace ptx;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float S_LIMIT = 1.2676506e30f;       // 2^100: rows above are redone with their maximum
constexpr float TERM_LEAST = 1.9721523e-31f;   // 2^-102: rows below V times that, too: V terms under 2^-126, which are 0, are 2^-24 of it
constexpr int CE_TILE = 256;
constexpr int CE_EPI = 8;
constexpr int CE_THREADS = (4 + CE_EPI) * 32;   // a control warpgroup (TMA, MMA, two idle warps) and two epilogue warpgroups
// An epilogue warp holds 128 accumulator columns: registers move from the control warpgroup to the epilogue's.  Launched with 168
// each (12 warps): 4 x 72 + 8 x 216 = 12 x 168.
constexpr int CE_REGS_CONTROL = 72, CE_REGS_EPI = 216;
static_assert(4 * CE_REGS_CONTROL + CE_EPI * CE_REGS_EPI <= 12 * 168, "setmaxnreg draws on the launch's registers");
constexpr int CE_CHUNK = 8;                    // float32: k-blocks between additions in registers

// MT row sub-tiles of 256 per pair tile: a stage holds this CTA's 128 rows of each and its half (128 rows) of B
template <int MT>
struct CeCfg {
    static constexpr int STAGES = MT == 2 ? 4 : 6;
    static constexpr int STAGE = (MT + 1) * SUB_BYTES;
    static constexpr int ROWS = MT * CE_TILE;
    static constexpr int SMEM = STAGES * STAGE + CE_EPI * 4096 + 1024;
    static_assert(SMEM <= 232448 - 512, "shared memory");
};

enum { EPI_SUM, EPI_EXP, EPI_PROB, EPI_SLOT, EPI_BF16, EPI_F32 };

struct CeArgs {
    const int32_t *count;         // rows left after gathering
    int64_t M, N;                 // output extents in tiles' terms (M ignored where the rows are counted on the device)
    int m_counted, k_counted;     // M, or the contraction, is *count
    int kbs;                      // 64-wide k-blocks per term
    int nterm;
    int a_off[6], b_off[6];       // column offsets of the parts a term multiplies
    int m_fast;
    int accumulate;               // EPI_SLOT: add to the slots instead of storing
    int tail, tail_parts;         // EPI_BF16 / EPI_F32: the last `tail` tiles are each cut into this many runs of k-blocks, stored in slots
    const float *off2, *scale, *tval;   // per row: exponent offset in powers of two; EPI_PROB: factor and the target's value
    const int32_t *tcol;          // per row: target column, -1 for none
    int32_t v0, ncols;            // first column of this piece, columns of it that exist
    float *partial;               // EPI_SUM / EPI_EXP: row sums, [2 per column tile][ld_partial]
    int64_t ld_partial;
    int part_cols;                // columns between the parts of the output (three parts: float32)
    int32_t *status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// L2 policies: what is read again soon (rows, the piece of the matrix) should outlive what streams past (E and P, several hundred MB)
__device__ __forceinline__ uint64_t l2_keep() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t l2_stream() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void tma_load_pair_hint(uint32_t smem_dst, const CUtensorMap *m, uint32_t cluster_bar, int32_t x, int32_t y, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(cluster_bar), "r"(x), "r"(y), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tma_store_hint(const CUtensorMap *m, uint32_t smem_src, int32_t x, int32_t y, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%2, %3}], [%1], %4;"
                 ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_src), "r"(x), "r"(y), "l"(policy) : "memory");
}
__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap *m, uint32_t smem_src, int32_t x, int32_t y) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_src), "r"(x), "r"(y) : "memory");
}

// ---- how the x-gradient's work is cut ---------------------------------------------------------------------------------------
// The row tiles of one 256-column tile each read the same rows of E, which is too large for L2: the `size` pairs of a group work
// on neighbouring column tiles of one row tile over the same run of k-blocks, so E crosses from memory once (R = 1024, 8192 rows,
// 25344 columns: 441 us when each pair had a run of its own).  Groups own equal runs of the (panel, k-block) sequence, a panel being
// a row tile and `size` column tiles.  Group g leaves its part of a panel in slot panel + g, which grows from each part to the next:
// (panels + groups) * size slots of one tile in float32 hold them all, whatever the number of rows turns out to be.
// Counts fit 32 bits (the entry points refuse more).
struct Cut {
    int total;                    // k-blocks of all panels
    int groups;                   // groups that take part: as many as get four k-blocks each
    int size, per_row, tiles_n;   // pairs per group, panels per row tile
    int KB;
    __host__ __device__ __forceinline__ Cut(int64_t rows, int64_t cols, int KB_, int pairs, int tile_rows) : KB(KB_) {
        tiles_n = (int)((cols + CE_TILE - 1) / CE_TILE);
        per_row = (tiles_n + 7) / 8;
        size = (tiles_n + per_row - 1) / per_row;
        total = (int)((rows + tile_rows - 1) / tile_rows) * per_row * KB;
        groups = pairs / size;      // pairs >= 8: every part of this GPU that the kernels run on has 16 SMs or more (ce_check)
        if (groups > total / 4) groups = total / 4 < 1 ? 1 : total / 4;
    }
    __host__ __device__ __forceinline__ int begin(int g) const { return (int)((int64_t)total * g / groups); }
    __host__ __device__ __forceinline__ int owner(int at) const { return (int)((((int64_t)at + 1) * groups + total - 1) / total - 1); }
    __host__ __device__ __forceinline__ int slots(int pairs) const { return (total / (KB ? KB : 1) + pairs / size) * size; }
};

struct WorkItem {
    int m, n, slot;               // slot < 0: the tile goes to the output itself
    int kb0, kb1;
};

// The sequence of work items of one pair; every role walks it by itself.
struct Walk {
    int tiles_m, tiles_n, next, end, step, whole, KB, parts, m_fast;
    int group, member, size, per_row;
    bool by_cut;
    __device__ __forceinline__ Walk(const CeArgs &a, bool by_cut_, int64_t rows, int kb_total, int pair, int pairs, int tile_rows)
        : KB(kb_total), m_fast(a.m_fast), by_cut(by_cut_) {
        tiles_m = (int)((rows + tile_rows - 1) / tile_rows);
        if (by_cut) {
            const Cut cut(rows, a.N, kb_total, pairs, tile_rows);
            tiles_n = cut.tiles_n;
            size = cut.size;
            per_row = cut.per_row;
            group = pair / size;
            member = pair % size;
            const bool in = group < cut.groups;
            next = in ? cut.begin(group) : 0;
            end = in ? cut.begin(group + 1) : 0;
        } else {
            tiles_n = (int)((a.N + CE_TILE - 1) / CE_TILE);
            step = pairs;
            parts = a.tail_parts;
            next = pair;
            whole = tiles_m * tiles_n - a.tail;
            end = whole + a.tail * parts;
        }
    }
    __device__ __forceinline__ bool take(WorkItem &w) {
        while (next < end) {
            if (!by_cut) {
                int tile = next;
                w.kb0 = 0;
                w.kb1 = KB;
                w.slot = -1;
                if (next >= whole) {
                    const int piece = (next - whole) % parts;
                    tile = whole + (next - whole) / parts;
                    w.slot = next - whole;
                    w.kb0 = KB * piece / parts;
                    w.kb1 = KB * (piece + 1) / parts;
                }
                w.m = m_fast ? tile % tiles_m : tile / tiles_n;
                w.n = m_fast ? tile / tiles_m : tile % tiles_n;
                next += step;
                return true;
            }
            const int panel = next / KB;
            w.kb0 = next - panel * KB;
            w.kb1 = end - next < KB - w.kb0 ? w.kb0 + end - next : KB;
            next += w.kb1 - w.kb0;
            w.m = panel / per_row;
            w.n = (panel % per_row) * size + member;
            w.slot = (panel + group) * size + member;
            if (w.n < tiles_n) return true;
        }
        return false;
    }
};

// 32 rows x 32 bf16 columns of a warp, from registers into a 2 KB staging box of 64-byte rows (the tiled copy's 64-byte swizzle:
// 16-byte piece p of row r goes to p ^ ((r >> 1) & 3), which spreads eight lanes over all banks)
__device__ __forceinline__ void stage_bf16(uint32_t box, int lane, const float *v) {
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
        uint32_t pk[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[ch * 8 + 2 * x], v[ch * 8 + 2 * x + 1]);
            pk[x] = *reinterpret_cast<const uint32_t *>(&h);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + (uint32_t)lane * 64u + (((uint32_t)ch ^ (((uint32_t)lane >> 1) & 3u)) << 4)), "r"(pk[0]), "r"(pk[1]),
                     "r"(pk[2]), "r"(pk[3]) : "memory");
    }
    fence_proxy_async_smem();
    __syncwarp();
}
// 32 rows x 32 float32 columns
__device__ __forceinline__ void stage_f32(uint32_t rowaddr, int lane, const float *v) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rowaddr + (uint32_t)((j ^ (lane & 7)) << 4)), "r"(__float_as_uint(v[4 * j])),
                     "r"(__float_as_uint(v[4 * j + 1])), "r"(__float_as_uint(v[4 * j + 2])), "r"(__float_as_uint(v[4 * j + 3])) : "memory");
    fence_proxy_async_smem();
    __syncwarp();
}

// PARTS 3: float32 operands (and MT 1, accumulators added up in registers).
template <int A_MN, int B_MN, int EPI, int PARTS, int MT>
__global__ void __launch_bounds__(CE_THREADS, 1)
ce_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
               const __grid_constant__ CUtensorMap tmap_d, const __grid_constant__ CUtensorMap tmap_slot, const __grid_constant__ CeArgs args) {
    using Cfg = CeCfg<MT>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr bool ADD = PARTS == 3;              // chunks of CE_CHUNK k-blocks, added in registers
    constexpr bool CUT = EPI == EPI_SLOT;
    static_assert(!ADD || MT == 1, "the registers hold one sub-tile");
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[STAGES], bar_free[STAGES], bar_tmem_full[2], bar_tmem_empty[2];
    __shared__ uint32_t tmem_holder;
    __shared__ int abort_flag;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t half = rank & 1;
    const bool leader = half == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);      // the even CTA's TMA thread; both CTAs' loads complete their bytes here
            mbar_init(smem_u32(&bar_free[s]), 1);      // one tcgen05.commit from the pair's MMA thread
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&bar_tmem_full[s]), 1);
            mbar_init(smem_u32(&bar_tmem_empty[s]), 2 * CE_EPI);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(&tmem_holder), TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_holder;
    volatile int *abortp = &abort_flag;
    pdl_launch_dependents();
    pdl_wait();

    const int64_t counted = (args.m_counted || args.k_counted) ? (int64_t)*args.count : 0;
    const int64_t rows = args.m_counted ? counted : args.M;
    const int kbs = args.k_counted ? (int)((counted + BK - 1) / BK) : args.kbs;
    Walk walk(args, CUT, rows, kbs * args.nterm, (int)(blockIdx.x >> 1), (int)(gridDim.x >> 1), Cfg::ROWS);
    WorkItem w;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CE_REGS_CONTROL));
        if (warp == 0) {
            // ------------------------------------------------------------------ TMA producer
            if (lane == 0) {
                prefetch_tmap(&tmap_a);
                prefetch_tmap(&tmap_b);
                const uint64_t pol_a = EPI <= EPI_PROB ? l2_keep() : l2_stream(), pol_b = EPI <= EPI_PROB ? l2_stream() : l2_keep();
                PipeState st;
                bool ok = true;
                while (ok && walk.take(w)) {
                    const int32_t m0 = (int32_t)(w.m * Cfg::ROWS + half * BM);
                    const int32_t n0 = (int32_t)(w.n * CE_TILE + half * BM);
                    int term = kbs ? w.kb0 / kbs : 0, kk = w.kb0 - term * kbs;
                    for (int kb = w.kb0; kb < w.kb1; ++kb) {
                        if (!mbar_wait_cluster(smem_u32(&bar_free[st.idx]), st.phase ^ 1, abortp)) {
                            raise_abort(abortp, args.status, RDB_STATUS_TIMEOUT_PRODUCER);
                            ok = false;
                            break;
                        }
                        const uint32_t fb = mapa(smem_u32(&bar_full[st.idx]), rank & ~1u);
                        if (leader) mbar_arrive_expect_tx(smem_u32(&bar_full[st.idx]), 2 * Cfg::STAGE);
                        const uint32_t sa = smem_base + st.idx * Cfg::STAGE, sb = sa + MT * SUB_BYTES;
                        const int32_t ax = args.a_off[term], bx = args.b_off[term], k0 = kk * BK;
#pragma unroll
                        for (int s = 0; s < MT; ++s) {
                            if (A_MN) {
#pragma unroll
                                for (int i = 0; i < BM / 64; ++i)
                                    tma_load_pair_hint(sa + s * SUB_BYTES + i * (64 * BK * 2), &tmap_a, fb, ax + m0 + s * CE_TILE + i * 64, k0, pol_a);
                            } else {
                                tma_load_pair_hint(sa + s * SUB_BYTES, &tmap_a, fb, ax + k0, m0 + s * CE_TILE, pol_a);
                            }
                        }
                        if (B_MN) {
#pragma unroll
                            for (int i = 0; i < BM / 64; ++i) tma_load_pair_hint(sb + i * (64 * BK * 2), &tmap_b, fb, bx + n0 + i * 64, k0, pol_b);
                        } else {
                            tma_load_pair_hint(sb, &tmap_b, fb, bx + k0, n0, pol_b);
                        }
                        st.advance<STAGES>();
                        if (++kk == kbs) { kk = 0; ++term; }
                    }
                }
                if (!ok) {
                    // gave up: let the loads already in flight land before the CTA may retire
                    const long long t0 = clock64();
                    while (clock64() - t0 < 4000000LL) {
                    }
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA issuer (even CTA of the pair)
            if (lane == 0 && leader) {
                constexpr uint32_t idesc = idesc_bf16_f32(2 * BM, CE_TILE, A_MN, B_MN);
                constexpr uint32_t desc_hi = smem_desc_hi_sw128(1024);
                constexpr uint32_t A_LBO = A_MN ? 64 * BK * 2 : 0, A_KSTEP = A_MN ? 2048 : UMMA_K * 2;
                constexpr uint32_t B_LBO = B_MN ? 64 * BK * 2 : 0, B_KSTEP = B_MN ? 2048 : UMMA_K * 2;
                const uint32_t peer = rank ^ 1u;
                bool ok = true;
                auto issue = [&](uint32_t stage, int sub, int acc, int k, bool fresh) {
                    const uint32_t sa = smem_base + stage * Cfg::STAGE;
                    const uint32_t a_lo = smem_desc_lo(sa + sub * SUB_BYTES, A_LBO), b_lo = smem_desc_lo(sa + MT * SUB_BYTES, B_LBO);
                    umma_bf16_pair(tmem_base + acc * CE_TILE, pack_desc(a_lo + ((k * A_KSTEP) >> 4), desc_hi),
                                   pack_desc(b_lo + ((k * B_KSTEP) >> 4), desc_hi), idesc, fresh ? 0u : 1u);
                };
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    if (!mbar_wait_cluster(bar, parity, abortp)) {
                        raise_abort(abortp, args.status, RDB_STATUS_TIMEOUT_MMA);
                        ok = false;
                    } else {
                        tc_fence_after_sync();
                    }
                    return ok;
                };
                auto commit_both = [&](uint32_t bar) {          // to the barrier of both CTAs
                    umma_commit_pair(bar);
                    umma_commit_pair(mapa(bar, peer));
                };
                if (MT == 1) {
                    PipeState st;
                    uint32_t it = 0;
                    while (ok && walk.take(w)) {
                        for (int c0 = w.kb0; c0 < w.kb1 && ok;) {
                            const int c1 = ADD && c0 + CE_CHUNK < w.kb1 ? c0 + CE_CHUNK : w.kb1;
                            const int acc = (int)(it & 1);
                            if (!wait(smem_u32(&bar_tmem_empty[acc]), ((it >> 1) & 1) ^ 1)) break;
                            for (int kb = c0; kb < c1; ++kb) {
                                if (!wait(smem_u32(&bar_full[st.idx]), st.phase)) break;
#pragma unroll
                                for (int k = 0; k < BK / UMMA_K; ++k) issue(st.idx, 0, acc, k, ((kb - c0) | k) == 0);
                                commit_both(smem_u32(&bar_free[st.idx]));
                                st.advance<STAGES>();
                            }
                            if (ok) commit_both(smem_u32(&bar_tmem_full[acc]));
                            ++it;
                            c0 = c1;
                        }
                    }
                } else {
                    // Two accumulators per tile.  While the epilogue still reads accumulator 1 of the tile before, the k-blocks that
                    // are staged already go to accumulator 0 alone (ahead of accumulator 1 by at most the ring); then both in turn:
                    // consecutive MMAs to one accumulator are a quarter slower.
                    PipeState st0, st1;
                    uint32_t it = 0;
                    while (ok && walk.take(w)) {
                        const int n = w.kb1 - w.kb0;
                        if (n == 0) continue;
                        const uint32_t par = (it & 1) ^ 1;
                        bool have1 = false;
                        int i0 = 0, i1 = 0;
                        while (i1 < n && ok) {
                            if (!have1 && (i0 - i1 == STAGES || i0 == n || mbar_try_wait_cluster(smem_u32(&bar_tmem_empty[1]), par))) {
                                if (!wait(smem_u32(&bar_tmem_empty[1]), par)) break;
                                have1 = true;
                            }
                            if (have1 && i1 < i0) {
#pragma unroll
                                for (int k = 0; k < BK / UMMA_K; ++k) issue(st1.idx, 1, 1, k, (i1 | k) == 0);
                                commit_both(smem_u32(&bar_free[st1.idx]));
                                st1.advance<STAGES>();
                                if (++i1 == n) commit_both(smem_u32(&bar_tmem_full[1]));
                                continue;
                            }
                            if (i0 == 0 && !wait(smem_u32(&bar_tmem_empty[0]), par)) break;
                            if (!wait(smem_u32(&bar_full[st0.idx]), st0.phase)) break;
                            const bool last = i0 == n - 1;
                            if (!have1 || last) {
#pragma unroll
                                for (int k = 0; k < BK / UMMA_K; ++k) issue(st0.idx, 0, 0, k, (i0 | k) == 0);
                                if (last) commit_both(smem_u32(&bar_tmem_full[0]));     // drained while accumulator 1 finishes
                                st0.advance<STAGES>();
                                ++i0;
                                continue;                                                // accumulator 1 catches up at the loop's top
                            }
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; ++k) {
                                issue(st0.idx, 0, 0, k, (i0 | k) == 0);
                                issue(st0.idx, 1, 1, k, (i0 | k) == 0);
                            }
                            commit_both(smem_u32(&bar_free[st0.idx]));
                            st0.advance<STAGES>();
                            st1.advance<STAGES>();
                            ++i0;
                            ++i1;
                        }
                        ++it;
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CE_REGS_EPI));
        // ------------------------------------------------------------------ epilogue: 8 warps, this CTA's 128 rows of a sub-tile
        const int ew = warp - 4;
        const int q = warp & 3;                      // TMEM lane quarter this warp may read
        const int cg = ew >> 2;                      // which 128 of the 256 columns
        const uint32_t leader_rank = rank & ~1u;
        const uint32_t stag = smem_base + STAGES * Cfg::STAGE + (uint32_t)ew * 4096u;
        const uint32_t rowaddr = stag + (uint32_t)lane * 128u;
        auto box_free = [&]() {                      // the last store from the staging box has read it
            if (lane == 0) bulk_wait_group_read0();
            __syncwarp();
        };
        // bf16: the box is two halves in turn, one being filled while the other is read; a group per use, empty or not
        uint32_t turn = 0;
        auto next_half = [&]() {
            if (lane == 0) bulk_wait_group_read1();
            __syncwarp();
            turn ^= 2048u;
            return stag + turn;
        };
        const uint64_t pol_e = l2_stream();
        uint32_t it = 0;
        bool ok = true;
        // this warp's 32 rows x 128 columns of the next accumulator, which goes back to the MMA thread
        auto drain = [&](float (&r)[128], int acc, uint32_t parity, bool add) {
            if (!mbar_wait_warp<true>(smem_u32(&bar_tmem_full[acc]), parity, abortp)) {
                raise_abort(abortp, args.status, RDB_STATUS_TIMEOUT_EPILOGUE);
                ok = false;
                return;
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * CE_TILE + cg * 128);
            if (add) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t t[32];
                    tmem_ld_32x32(taddr + b * 32, t);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[b * 32 + j] += __uint_as_float(t[j]);
                }
            } else {
                uint32_t(&t)[128] = reinterpret_cast<uint32_t(&)[128]>(r);
#pragma unroll
                for (int b = 0; b < 4; ++b) tmem_ld_32x32(taddr + b * 32, reinterpret_cast<uint32_t(&)[32]>(t[b * 32]));
                tmem_ld_wait();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(mapa(smem_u32(&bar_tmem_empty[acc]), leader_rank));
        };
        while (ok && walk.take(w)) {
            const int64_t n0 = (int64_t)w.n * CE_TILE + cg * 128;
#pragma unroll 1
            for (int s = 0; s < MT && ok; ++s) {
                const int64_t row_w = (int64_t)w.m * Cfg::ROWS + s * CE_TILE + half * BM + q * 32;
                float off = 0.0f, scale = 0.0f, tval = 0.0f;
                int t_rel = -1;
                if (EPI <= EPI_PROB) {               // the rows' numbers are fetched while the tile is being multiplied
                    off = args.off2[row_w + lane];
                    t_rel = args.tcol[row_w + lane] - args.v0 - (int)n0;
                    if (EPI == EPI_PROB) { scale = args.scale[row_w + lane]; tval = args.tval[row_w + lane]; }
                }
                float r[128];
                if (EPI >= EPI_BF16 && w.kb0 == w.kb1) {   // nothing to contract
#pragma unroll
                    for (int j = 0; j < 128; ++j) r[j] = 0.0f;
                } else if (MT == 2) {
                    drain(r, s, it & 1, false);
                } else if (!ADD) {
                    drain(r, (int)(it & 1), (it >> 1) & 1, false);
                    ++it;
                } else {
#pragma unroll
                    for (int j = 0; j < 128; ++j) r[j] = 0.0f;
                    for (int c0 = w.kb0; c0 < w.kb1 && ok; c0 += CE_CHUNK, ++it) drain(r, (int)(it & 1), (it >> 1) & 1, true);
                }
                if (!ok) break;
                if (EPI <= EPI_PROB) {
                    float sum = 0.0f;
#pragma unroll
                    for (int hb = 0; hb < 2; ++hb) {
                        float *e = r + hb * 64;
                        const int c0 = (int)n0 + hb * 64, tr = t_rel - hb * 64;
#pragma unroll
                        for (int j = 0; j < 64; ++j) e[j] = ex2(__fmaf_rn(e[j], LOG2E, -off));
                        if (c0 + 64 > args.ncols) {
#pragma unroll
                            for (int j = 0; j < 64; ++j) e[j] = c0 + j < args.ncols ? e[j] : 0.0f;
                        }
                        if (EPI == EPI_PROB) {
#pragma unroll
                            for (int j = 0; j < 64; ++j) e[j] *= scale;
                            if (row_w + 32 > rows) {             // padding, which the weight gradient contracts with: 0 even against an infinite weight
#pragma unroll
                                for (int j = 0; j < 64; ++j) e[j] = row_w + lane < rows ? e[j] : 0.0f;
                            }
                        }
                        if (__any_sync(0xffffffffu, (unsigned)tr < 64u)) {      // a target among these columns: left out of the sum
                            const float tv = EPI == EPI_PROB ? tval : 0.0f;
#pragma unroll
                            for (int j = 0; j < 64; ++j) e[j] = j == tr ? tv : e[j];
                        }
                        if (EPI != EPI_PROB) {
                            float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
#pragma unroll
                            for (int j = 0; j < 64; j += 4) { a0 += e[j]; a1 += e[j + 1]; a2 += e[j + 2]; a3 += e[j + 3]; }
                            sum += (a0 + a1) + (a2 + a3);
                        }
                        if (EPI != EPI_SUM) {
#pragma unroll
                            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                                for (int b = 0; b < 2; ++b) {
                                    const uint32_t box = next_half();
                                    stage_bf16(box, lane, e + b * 32);
                                    if (p + 1 < PARTS) {
#pragma unroll
                                        for (int j = b * 32; j < b * 32 + 32; ++j) e[j] -= __bfloat162float(__float2bfloat16_rn(e[j]));
                                    }
                                    if (lane == 0) {
                                        tma_store_hint(&tmap_d, box, p * args.part_cols + c0 + b * 32, (int32_t)row_w, pol_e);
                                        bulk_commit_group();
                                    }
                                }
                            }
                        }
                    }
                    if (EPI != EPI_PROB) args.partial[(w.n * 2 + cg) * args.ld_partial + row_w + lane] = sum;
                } else if (EPI == EPI_BF16 && w.slot < 0) {
#pragma unroll
                    for (int cb = 0; cb < 4; ++cb) {
                        const uint32_t box = next_half();
                        stage_bf16(box, lane, r + cb * 32);
                        const int64_t c0 = n0 + cb * 32;
                        if (lane == 0) {
                            if (row_w < rows && c0 < args.N) tma_store_2d(&tmap_d, box, (int32_t)c0, (int32_t)row_w);
                            bulk_commit_group();
                        }
                    }
                } else {
                    // float32 boxes, to the output or to a slot
#pragma unroll
                    for (int cb = 0; cb < 4; ++cb) {
                        box_free();
                        stage_f32(rowaddr, lane, r + cb * 32);
                        if (lane == 0) {
                            const int64_t c0 = n0 + cb * 32;
                            if (w.slot >= 0) {
                                const int32_t x = cg * 128 + cb * 32, y = (int32_t)(w.slot * Cfg::ROWS + s * CE_TILE + half * BM + q * 32);
                                if (EPI == EPI_SLOT && args.accumulate) tma_reduce_add_2d(&tmap_slot, stag, x, y);
                                else tma_store_2d(&tmap_slot, stag, x, y);
                                bulk_commit_group();
                            } else if (c0 < args.N && row_w < rows) {
                                tma_store_2d(&tmap_d, stag, (int32_t)c0, (int32_t)row_w);
                                bulk_commit_group();
                            }
                        }
                    }
                }
            }
            if (MT == 2 && w.kb0 != w.kb1) ++it;
        }
        if (EPI != EPI_SUM && lane == 0) bulk_wait_group0();     // all output written before the CTA retires
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // no CTA retires (or frees TMEM) while its peer may still use it
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// Output rows of the tiles whose contraction was cut (CeArgs::tail): their parts, added in order.  A block takes four rows, a thread
// four columns of one.
template <typename T>
__global__ void __launch_bounds__(256) ce_tail_kernel(T *__restrict__ out, int64_t ldo, const float *__restrict__ slots, int64_t M, int64_t N,
                                                      int first, int parts, int tile_rows) {
    pdl_launch_dependents();
    pdl_wait();
    const int tiles_n = (int)((N + CE_TILE - 1) / CE_TILE);
    const int r4 = tile_rows / 4, i = blockIdx.x / r4;
    const int r = (blockIdx.x % r4) * 4 + (threadIdx.x >> 6), cl = (threadIdx.x & 63) * 4;
    const int tile = first + i;
    const int64_t row = (int64_t)(tile / tiles_n) * tile_rows + r, col = (int64_t)(tile % tiles_n) * CE_TILE + cl;
    if (row >= M || col >= N) return;
    const float *p = slots + ((int64_t)i * parts * tile_rows + r) * CE_TILE + cl;
    float4 v = *reinterpret_cast<const float4 *>(p);
#pragma unroll 4
    for (int k = 1; k < parts; ++k) {
        const float4 u = *reinterpret_cast<const float4 *>(p + (int64_t)k * tile_rows * CE_TILE);
        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
    T *o = out + row * ldo + col;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < N) o[e] = from_f32<T>(f[e]);
}

// rows of a padded matrix to a dense one whose rows start on no vector boundary
template <typename T>
__global__ void __launch_bounds__(256) ce_copy_kernel(T *__restrict__ dst, const T *__restrict__ src, int64_t rows, int64_t cols, int64_t ld) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    for (int64_t c = threadIdx.x & 63; c < cols; c += 64) dst[r * cols + c] = src[r * ld + c];
}

// ================================================================================================
// rows
// ================================================================================================
// Positions of the rows that count, in order: idx[compact] = row, map[row] = compact or -1.  One block; the losses (zero_*, may be
// null) are cleared at ignored rows, the ticket of the kernel that sums them is reset.
__global__ void __launch_bounds__(1024) ce_rows_kernel(const int64_t *__restrict__ target, int64_t T, int64_t ignore, int use_ignore,
                                                       int32_t *__restrict__ idx, int32_t *__restrict__ map, int32_t *__restrict__ count,
                                                       float *__restrict__ zero_a, float *__restrict__ zero_b, float *__restrict__ zero_c,
                                                       float *__restrict__ count_f, uint32_t *__restrict__ ticket, int2 *__restrict__ parts,
                                                       int64_t cols, int KB, int pairs, int tile_rows) {
    constexpr int PER = 8;
    __shared__ int warp_sum[2][32];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int base = 0, turn = 0;
    for (int64_t b = 0; b < T; b += 1024 * PER, turn ^= 1) {
        const int64_t i0 = b + warp * (32 * PER) + lane;        // a warp takes 256 rows in a stretch, a lane every 32nd
        int64_t t[PER];
        unsigned keep[PER];
        int n = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) t[k] = i0 + k * 32 < T ? target[i0 + k * 32] : 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            keep[k] = __ballot_sync(0xffffffffu, i0 + k * 32 < T && !(use_ignore && t[k] == ignore));
            n += __popc(keep[k]);
        }
        if (lane == 0) warp_sum[turn][warp] = n;
        __syncthreads();
        int ws = warp_sum[turn][lane];               // every warp scans the warps' sums itself
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, ws, o);
            if (lane >= o) ws += y;
        }
        const int before = __shfl_sync(0xffffffffu, ws, warp) - n;
        int at = base + before;
        base += __shfl_sync(0xffffffffu, ws, 31);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int64_t i = i0 + k * 32;
            const int j = at + __popc(keep[k] & ((1u << lane) - 1u));
            at += __popc(keep[k]);
            if (i < T) {
                const bool ok = (keep[k] >> lane) & 1u;
                map[i] = ok ? j : -1;
                if (ok) idx[j] = (int32_t)i;
                else {
                    if (zero_a) zero_a[i] = 0.0f;
                    if (zero_b) zero_b[i] = 0.0f;
                    if (zero_c) zero_c[i] = 0.0f;
                }
            }
        }
    }
    // where the parts of each panel of the x-gradient begin and how many there are, for the kernels that add them
    if (parts) {
        const Cut cut(base, cols, KB, pairs, tile_rows);
        const int panels = (base + tile_rows - 1) / tile_rows * cut.per_row;
        for (int p = threadIdx.x; p < panels; p += 1024) {
            const int lo = cut.owner(p * KB);
            parts[p] = make_int2(lo, cut.owner((p + 1) * KB - 1) - lo + 1);
        }
    }
    if (threadIdx.x == 0) {
        *count = base;
        *ticket = 0;
        if (count_f) *count_f = (float)base;
    }
}

// The matrix a row's target selects: stored, or noise.
struct Vocab {
    const void *w;        // null: noise
    int64_t ldw;
    uint32_t seed, row0;
};

template <typename T> __device__ __forceinline__ float vocab_at(const Vocab &v, int64_t row, int64_t col) {
    if (v.w) return to_f32<T>(reinterpret_cast<const T *>(v.w)[row * v.ldw + col]);
    return to_f32<T>(from_f32<T>(sq5_to_float(sq5_bits(v.row0 + (uint32_t)row, (uint32_t)col, v.seed))));
}

// The first of several bf16 parts: a finite value beyond bf16's largest (float32's lowest, as masks have it) must not round to infinity.
__device__ __forceinline__ float first_part(float v) {
    constexpr float MOST = 3.38953139e38f;
    return fabsf(v) > MOST && fabsf(v) <= 3.402823466e38f ? copysignf(MOST, v) : v;
}
template <int PARTS> __device__ __forceinline__ void split_store(__nv_bfloat16 *dst, int64_t part_cols, int64_t c, float v) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        const __nv_bfloat16 h = __float2bfloat16_rn(PARTS > 1 && p == 0 ? first_part(v) : v);
        dst[p * part_cols + c] = h;
        v -= __bfloat162float(h);
    }
}

struct CeRowArgs {
    const void *x;
    int64_t ldx, T, R, V;
    const int64_t *target;
    const int32_t *idx, *count;
    __nv_bfloat16 *a;             // gathered rows [rows, PARTS * part_cols]
    int64_t lda, part_cols;
    float *off2, *lt, *dist, *scale, *tval;
    float spread;                 // mean of the largest of V standard normal values
    int32_t *tcol;
    // backward
    const float *dloss;           // null: forward
    const float *lse, *loss;
    int reduction;
    int tile_rows;
};

// eight consecutive elements, 16-byte aligned for bf16 and 32-byte for float32
__device__ __forceinline__ void load_f8(float (&f)[8], const __nv_bfloat16 *p) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) { f[2 * k] = __low2float(h[k]); f[2 * k + 1] = __high2float(h[k]); }
}
__device__ __forceinline__ void load_f8(float (&f)[8], const float *p) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ uint4 pack_f8(const float (&f)[8]) {
    uint4 v;
    uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return v;
}
template <int PARTS> __device__ __forceinline__ void split_store8(__nv_bfloat16 *dst, int64_t part_cols, float (&f)[8]) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        float h[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = PARTS > 1 && p == 0 ? first_part(f[k]) : f[k];
        const uint4 v = pack_f8(h);
        *reinterpret_cast<uint4 *>(dst + p * part_cols) = v;
        if (p + 1 < PARTS) {
            float g[8];
            load_f8(g, reinterpret_cast<const __nv_bfloat16 *>(&v));
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] -= g[k];
        }
    }
}
template <typename T> __device__ __forceinline__ bool rows_aligned(const void *base, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
}

// Sums over the warp of N values per lane (N a power of two): lane i gets that of value i % N.  Each step halves what a lane keeps.
template <int N> __device__ __forceinline__ float warp_sums(float (&v)[N], int lane) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if (i < o) {
                const float give = upper ? v[i] : v[i + o];
                const float got = __shfl_xor_sync(0xffffffffu, give, o);
                v[i] = (upper ? v[i + o] : v[i]) + got;
            }
        }
    }
    float l = v[0];
#pragma unroll
    for (int o = N; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return l;
}

// Where the largest logit of a row over a stored matrix will lie, from SAMPLES vocabulary rows spread evenly (the target's left out; exact
// where there are no more): the logits' mean plus `spread` deviations, and at least the largest one seen.  `sigma` is the deviation that the row's
// length gives, which holds for logits that are independent with mean 0 (over a noise matrix they are).  Where the matrix's rows share a component,
// as trained ones do, it is too large, for that lengthens all of them and spreads none: so the samples' mean counts where it is four standard errors
// off 0, and their deviation (which 32 samples know to 13 %) where sigma is 1.6 times as large, or half.  Four samples are enough where even sigma,
// four standard errors above their mean, stays below `enough`: minus infinity then.  By a warp.  8192 rows of 768, V = 50257, loss, ms, by the length
// alone -> with samples: logits of deviation 3 about -100, or of deviation 10 about 60 beside a common component that the rows of x do not have, 61
// (every row was redone) -> 0.53; deviation 20 about 60 35 -> 0.54, about -300 61 -> 10; independent logits of deviation 2 0.49 -> 0.49, of deviation 8
// to 40 0.49 -> 0.51 to 0.55.
constexpr int SAMPLES = 32;
template <typename T>
__device__ __noinline__ float sampled_top(const CeRowArgs &a, const Vocab &voc, const T *src, int64_t target, float sigma, float enough, int lane) {
    const bool vec = rows_aligned<T>(a.x, a.ldx) && rows_aligned<T>(voc.w, voc.ldw);
    const int64_t done = vec ? a.R / 8 * 8 : 0;
    auto sample = [&](int k) -> int64_t {         // in the order 0, 1/2, 1/4, 3/4, ...
        if (a.V <= SAMPLES) return k < a.V ? k : a.V - 1;
        return (int64_t)(2 * (__brev((unsigned)k) >> 27) + 1) * a.V / (2 * SAMPLES);
    };
    static_assert(SAMPLES == 32, "one per lane, five bits");
    const bool on = lane < a.V && sample(lane) != target;
    // mean and deviation of the samples of the lanes in `who`
    auto spread_of = [&](float l, bool who, float &mean, float &dev) {
        const float n = (float)__popc(__ballot_sync(0xffffffffu, who));
        mean = who ? l : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
        mean /= n;
        dev = who ? (l - mean) * (l - mean) : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) dev += __shfl_xor_sync(0xffffffffu, dev, o);
        dev = sqrtf(dev / (n - 1.0f));
        return n;
    };
    float mean, dev;
    float mine = 0.0f;                            // lane k holds the logit of sample k
    for (int k0 = 0; k0 < SAMPLES && k0 < a.V; k0 += 4) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t c = lane * 8; c < done; c += 256) {
            float f[8], w[8];
            load_f8(f, src + c);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t v = sample(k0 + q);
                load_f8(w, reinterpret_cast<const T *>(voc.w) + v * voc.ldw + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[q] = fmaf(f[e], w[e], acc[q]);
            }
        }
        for (int64_t c = done + lane; c < a.R; c += 32) {
            const float f = to_f32<T>(src[c]);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = fmaf(f, to_f32<T>(reinterpret_cast<const T *>(voc.w)[sample(k0 + q) * voc.ldw + c]), acc[q]);
        }
        const float l = warp_sums(acc, lane);
        if (lane / 4 == k0 / 4) mine = l;
        if (k0 == 0 && a.V > SAMPLES) {
            spread_of(mine, on && lane < 4, mean, dev);
            if (dev < 2.0f * sigma && mean + (a.spread + 2.0f) * sigma < enough) return -INFINITY;
        }
    }
    float most = on ? mine : -INFINITY;
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (a.V <= SAMPLES) return most;
    const float n = spread_of(mine, on, mean, dev);
    if (fabsf(mean) * sqrtf(n) < 4.0f * dev) mean = 0.0f;
    if (sigma > 1.6f * dev) sigma = 1.3f * dev;
    else if (dev > 2.0f * sigma) sigma = dev;
    return fmaxf(most, mean + a.spread * sigma);
}

// One warp per gathered row: the row in bf16 parts, its target's logit (forward), or exponent offset, factor and target value of
// the probabilities (backward).  Rows up to the tile's end are zeros that contribute nothing anywhere.
template <typename T, int PARTS>
__global__ void __launch_bounds__(256, 4) ce_gather_kernel(const __grid_constant__ CeRowArgs a, const __grid_constant__ Vocab voc) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t n = *a.count;
    if (j >= (n + a.tile_rows - 1) / a.tile_rows * a.tile_rows) return;
    __nv_bfloat16 *dst = a.a + j * a.lda;
    if (j >= n) {
        for (int64_t c = lane * 8; c < a.lda; c += 256) *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0, 0, 0, 0);
        if (lane == 0) {
            a.off2[j] = INFINITY;
            a.tcol[j] = -1;
            if (a.dloss) { a.scale[j] = 0.0f; a.tval[j] = 0.0f; }
        }
        return;
    }
    const int64_t row = a.idx[j];
    const int64_t t = a.target[row];
    const bool known = t >= 0 && t < a.V;
    const bool dot_it = !a.dloss && known;
    const T *src = reinterpret_cast<const T *>(a.x) + row * a.ldx;
    float dot = 0.0f, xx = 0.0f, ww = 0.0f;
    // the same order of additions whether or not the operands start on vector boundaries
    const bool vx = rows_aligned<T>(a.x, a.ldx), vw = voc.w && rows_aligned<T>(voc.w, voc.ldw);
    const T *wrow = reinterpret_cast<const T *>(voc.w) + (voc.w && dot_it ? t * voc.ldw : 0);
    const Sq5Lin lin = sq5_lin_rows(voc.seed, voc.row0 + (uint32_t)t, 0u);
    const int64_t done = a.R / 8 * 8;
#pragma unroll 4
    for (int64_t c = lane * 8; c < done; c += 256) {
        float f[8], w[8];
        if (vx) load_f8(f, src + c);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = to_f32<T>(src[c + k]);
        }
        if (dot_it) {
            if (vw) load_f8(w, wrow + c);
            else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    w[k] = voc.w ? to_f32<T>(wrow[c + k]) : to_f32<T>(from_f32<T>(sq5_to_float(sq5_tail(lin.base + ((uint32_t)c + k) * lin.sk))));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                dot = fmaf(f[k], w[k], dot);
                xx = fmaf(f[k], f[k], xx);
                ww = fmaf(w[k], w[k], ww);
            }
        }
        split_store8<PARTS>(dst + c, a.part_cols, f);
    }
    for (int64_t c = done + lane; c < a.part_cols; c += 32) {
        const float v = c < a.R ? to_f32<T>(src[c]) : 0.0f;
        split_store<PARTS>(dst, a.part_cols, c, v);
        if (dot_it && c < a.R) {
            const float w = vocab_at<T>(voc, t, c);
            dot = fmaf(v, w, dot);
            xx = fmaf(v, v, xx);
            ww = fmaf(w, w, ww);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        xx += __shfl_xor_sync(0xffffffffu, xx, o);
        ww += __shfl_xor_sync(0xffffffffu, ww, o);
    }
    float d = 0.0f;
    if (!a.dloss) {                                   // (the whole warp holds the sums)
        if (!known) dot = NAN;                        // a target outside the vocabulary: the row's loss says so
        const float sigma = sqrtf(xx) * sqrtf(ww / (float)a.R), top = sigma * a.spread;
        if (!voc.w) d = top - dot;
        // (stored: where the logits' mean is not 0, the target's may be high and the largest far above it all the same)
        else if ((top - dot >= 40.0f || sigma * (a.spread + 3.0f) >= 60.0f) && top < 1e6f) d = sampled_top<T>(a, voc, src, t, sigma, dot + 60.0f, lane) - dot;
        if (!(d >= 40.0f && d < 1e6f)) d = 0.0f;
    }
    if (lane == 0) {
        a.tcol[j] = known ? (int32_t)t : -1;
        if (!a.dloss) {
            a.lt[j] = dot;
            a.dist[j] = d;
            a.off2[j] = (dot + d) * LOG2E;
        } else {
            const float g = a.reduction == RDB_CE_NONE ? a.dloss[row] : a.reduction == RDB_CE_MEAN ? a.dloss[0] / (float)n : a.dloss[0];
            a.off2[j] = a.lse[row] * LOG2E;
            a.scale[j] = g;
            a.tval[j] = g * expm1f(-a.loss[row]);     // softmax - 1 at the target, without a difference
        }
    }
}

// rows of the matrix in bf16 parts, zero between R and part_cols; a thread takes eight columns of a row
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) ce_split_kernel(__nv_bfloat16 *__restrict__ dst, int64_t ldd, int64_t part_cols, int64_t rows, int64_t R,
                                                       int64_t v0, Vocab voc) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t per = (uint32_t)(part_cols / 8);
    const int64_t total = rows * per;
    const bool vec = voc.w && rows_aligned<T>(voc.w, voc.ldw);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i >> 32 ? i / per : (uint32_t)i / per;
        const int64_t c = (i - r * per) * 8;
        float f[8];
        if (vec && c + 8 <= R) {
            load_f8(f, reinterpret_cast<const T *>(voc.w) + (v0 + r) * voc.ldw + c);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = c + k < R ? vocab_at<T>(voc, v0 + r, c + k) : 0.0f;
        }
        split_store8<PARTS>(dst + r * ldd + c, part_cols, f);
    }
}

// ================================================================================================
// finishing
// ================================================================================================
// The parts of row j, column tile n of the x-gradient: `first` is column 0 of the first part, `step` elements lie between the parts.
struct SlotRow {
    float *first;
    int64_t step;
    int n;
    __device__ __forceinline__ SlotRow(float *slots, const int2 *parts, int tiles_n, int tile_rows, int64_t j, int nt) {
        const int per_row = (tiles_n + 7) / 8, size = (tiles_n + per_row - 1) / per_row;      // as Cut has them
        const int m = (int)j / tile_rows, panel = m * per_row + nt / size;
        const int2 p = parts[panel];
        first = slots + (((int64_t)(panel + p.x) * size + nt % size) * tile_rows + (j - (int64_t)m * tile_rows)) * CE_TILE;
        step = (int64_t)size * tile_rows * CE_TILE;
        n = p.y;
    }
};

// What is known of the rows once all their logits have been seen.
struct CeSumArgs {
    CeRowArgs rows;
    Vocab voc;
    const float *partial;
    int64_t ld_partial;
    int nparts;
    float *s;                     // per gathered row: s, or -1: its gradient is finished
    float *lse, *loss_rows, *loss_rows2;
    float *slots;                 // null: no gradient
    const int2 *parts;
    float *loss;                  // null: no total
    int mean;
    float least;                  // of s, where it is relative to an estimate
    uint32_t *ticket;             // zero at the start
};

// add one logit to a running (maximum, sum relative to it)
__device__ __forceinline__ void online(float &m, float &s, float l) {
    if (l > m) {
        s = s * ex2((m - l) * LOG2E) + 1.0f;
        m = l;
    } else if (l == m) {
        s += l == -INFINITY ? 0.0f : 1.0f;    // a difference of two infinities would be NaN
    } else {
        s += ex2((l - m) * LOG2E);
    }
}
__device__ __forceinline__ void online_join(float &m, float &s, float m2, float s2) {
    const float mm = fmaxf(m, m2);
    s = (m == mm ? s : s * ex2((m - mm) * LOG2E)) + (m2 == mm ? s2 : s2 * ex2((m2 - mm) * LOG2E));
    m = mm;
}

// log(1 + s e^up): the loss of a row whose other logits have a largest one `up` above the target's and a sum s relative to that
__device__ __forceinline__ float loss_above(float up, float s) {
    return s == 0.0f ? 0.0f : up < 60.0f ? log1pf(s * expf(up)) : up + logf(s + expf(-up));
}

// Rows whose sum left float32's range: their logits once more on CUDA cores, first the maximum and the sum relative to it, then, with
// slots, the gradient itself, which goes to a row's first slot.  By the whole block (512 threads), for up to FAR of its rows at a time
// (`far`: bit r is row j0 + r): a warp multiplies FAR_ROWS rows of the matrix with all of them.  Bound by what one SM can load
// (stored) or hash (noise).  Among 8192 rows of 768, V = 50257, the call takes, ms: stored, loss, no such row 0.5, one 3.8, every eighth 8.0, the first 1024 in
// a row 59 (one row at a time, a logit per warp: 25 and 84 for the first two); noise, loss and gradient 1.0, 16, 53, 412.
constexpr int FAR = 2, FAR_ROWS = 4, FAR_COLS = 4;

template <typename T>
__device__ __noinline__ void ce_far_rows(const CeSumArgs &g, int64_t j0, unsigned far) {
    __shared__ float2 sh_ms[16][FAR];
    __shared__ float3 sh_ref[FAR];                 // the larger of target's and others' largest logit, log-sum-exp above it, loss
    __shared__ __align__(16) float sh_p[16 * FAR_ROWS][FAR];
    const CeRowArgs &a = g.rows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = (int)a.R;
    const int n = __popc(far) < FAR ? __popc(far) : FAR;
    int64_t j[FAR];
    const T *x[FAR];
    int64_t target[FAR];
    unsigned left = far;
#pragma unroll
    for (int t = 0; t < FAR; ++t) {                // past the last one: the last one again, whose results nothing reads
        j[t] = j0 + __ffs(left) - 1;
        if (t + 1 < n) left &= left - 1;
        const int64_t row = a.idx[j[t]];
        x[t] = reinterpret_cast<const T *>(a.x) + row * a.ldx;
        target[t] = a.target[row];
    }
    constexpr int PAIRS = FAR_ROWS * FAR;
    static_assert(FAR == 2, "two rows");
    const int my_row = lane % PAIRS / FAR, my_t = lane % FAR;      // whose logit the lane gets
    const int64_t my_target = target[my_t ? 1 : 0];
    constexpr int W = 16 / sizeof(T);              // elements of a 16-byte load
    const bool vec = g.voc.w && rows_aligned<T>(g.voc.w, g.voc.ldw) && rows_aligned<T>(a.x, a.ldx);
    const int whole = vec ? R / W * W : 0;
    // logits of matrix rows v0 .. v0 + 3 (rows past the end: the last one's)
    auto logits = [&](int64_t v0) {
        float acc[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) acc[i] = 0.0f;
        if (g.voc.w) {
            const T *w[FAR_ROWS];
#pragma unroll
            for (int r = 0; r < FAR_ROWS; ++r) w[r] = reinterpret_cast<const T *>(g.voc.w) + (v0 + r < a.V ? v0 + r : a.V - 1) * g.voc.ldw;
#pragma unroll 2
            for (int c = lane * W; c < whole; c += 32 * W) {
                uint4 u[FAR_ROWS];
#pragma unroll
                for (int r = 0; r < FAR_ROWS; ++r) u[r] = __ldg(reinterpret_cast<const uint4 *>(w[r] + c));
#pragma unroll
                for (int t = 0; t < FAR; ++t) {
                    const uint4 f = __ldg(reinterpret_cast<const uint4 *>(x[t] + c));
#pragma unroll
                    for (int e = 0; e < W; ++e)
#pragma unroll
                        for (int r = 0; r < FAR_ROWS; ++r)
                            acc[r * FAR + t] = fmaf(to_f32<T>(reinterpret_cast<const T *>(&f)[e]), to_f32<T>(reinterpret_cast<const T *>(&u[r])[e]), acc[r * FAR + t]);
                }
            }
#pragma unroll 2
            for (int c = whole + lane; c < R; c += 32)
#pragma unroll
                for (int r = 0; r < FAR_ROWS; ++r) {
                    const float f = to_f32<T>(w[r][c]);
#pragma unroll
                    for (int t = 0; t < FAR; ++t) acc[r * FAR + t] = fmaf(to_f32<T>(x[t][c]), f, acc[r * FAR + t]);
                }
        } else {
            uint32_t h = sq5_lin_rows(g.voc.seed, g.voc.row0 + (uint32_t)v0, (uint32_t)lane).base;
#pragma unroll 2
            for (int c = lane; c < R; c += 32, h += 32u * SQ5_N1) {
                float f[FAR];
#pragma unroll
                for (int t = 0; t < FAR; ++t) f[t] = to_f32<T>(x[t][c]);
#pragma unroll
                for (int r = 0; r < FAR_ROWS; ++r) {
                    const float w = to_f32<T>(from_f32<T>(sq5_to_float(sq5_tail(h + (uint32_t)r * (SQ5_PRIME * SQ5_N1)))));
#pragma unroll
                    for (int t = 0; t < FAR; ++t) acc[r * FAR + t] = fmaf(f[t], w, acc[r * FAR + t]);
                }
            }
        }
        return warp_sums(acc, lane);
    };
    float m = -INFINITY, s = 0.0f;                 // over the columns other than the target
    for (int64_t v0 = warp * FAR_ROWS; v0 < a.V; v0 += 16 * FAR_ROWS) {
        const float l = logits(v0);
        if (lane < PAIRS && v0 + my_row < a.V && v0 + my_row != my_target) online(m, s, l);
    }
#pragma unroll
    for (int o = FAR; o < 32; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        online_join(m, s, m2, s2);
    }
    __syncthreads();                               // the rows before are done with the arrays
    if (lane < FAR) sh_ms[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < n) {
        const int t = threadIdx.x;
        float2 r = sh_ms[0][t];
        for (int k = 1; k < 16; ++k) online_join(r.x, r.y, sh_ms[k][t].x, sh_ms[k][t].y);
        const int64_t jt = j[t ? 1 : 0], row = a.idx[jt];
        const float lt = a.lt[jt], up = r.x - lt, l = loss_above(up, r.y);
        const float ref = up > 0.0f ? r.x : lt, rest = up > 0.0f ? logf(r.y + expf(-up)) : l;
        g.loss_rows[row] = l;
        if (g.loss_rows2) g.loss_rows2[row] = l;
        g.lse[row] = ref + rest;
        g.s[jt] = -1.0f;
        sh_ref[t] = make_float3(ref, rest, l);
    }
    if (!g.slots) return;
    __syncthreads();
    const float3 my_ref = sh_ref[my_t < n ? my_t : n - 1];
    const int tiles_n = (int)((a.R + CE_TILE - 1) / CE_TILE);
    for (int c0 = 0; c0 < R; c0 += 512 * FAR_COLS) {              // so many columns at a time, FAR_COLS per thread
        float acc[FAR_COLS][FAR];
#pragma unroll
        for (int k = 0; k < FAR_COLS; ++k) {
            const int c = c0 + k * 512 + (int)threadIdx.x;
#pragma unroll
            for (int t = 0; t < FAR; ++t) {
                acc[k][t] = c < R ? expm1f(-sh_ref[t < n ? t : n - 1].z) * vocab_at<T>(g.voc, target[t], c) : 0.0f;
            }
        }
        for (int64_t v0 = 0; v0 < a.V; v0 += 16 * FAR_ROWS) {
            const int64_t v = v0 + warp * FAR_ROWS + my_row;
            if (v0 + warp * FAR_ROWS < a.V) {
                const float l = logits(v0 + warp * FAR_ROWS);
                if (lane < PAIRS) sh_p[warp * FAR_ROWS + my_row][my_t] = v < a.V && v != my_target ? expf((l - my_ref.x) - my_ref.y) : 0.0f;
            }
            __syncthreads();
            const int rows = a.V - v0 < 16 * FAR_ROWS ? (int)(a.V - v0) : 16 * FAR_ROWS;
#pragma unroll 1
            for (int k = 0; k < rows; ++k) {
                const float2 p = *reinterpret_cast<const float2 *>(sh_p[k]);
                if (p.x == 0.0f && p.y == 0.0f) continue;
#pragma unroll
                for (int q = 0; q < FAR_COLS; ++q) {
                    const int c = c0 + q * 512 + (int)threadIdx.x;
                    if (c < R) {
                        const float w = vocab_at<T>(g.voc, v0 + k, c);
                        acc[q][0] = fmaf(p.x, w, acc[q][0]);
                        acc[q][1] = fmaf(p.y, w, acc[q][1]);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int q = 0; q < FAR_COLS; ++q) {
            const int c = c0 + q * 512 + (int)threadIdx.x;
            if (c >= R) continue;
#pragma unroll
            for (int t = 0; t < FAR; ++t)
                if (t < n) SlotRow(g.slots, g.parts, tiles_n, a.tile_rows, j[t], c / CE_TILE).first[c % CE_TILE] = acc[q][t];
        }
    }
}

// s, log-sum-exp and loss of 32 rows per block: sixteen threads per row add every sixteenth partial sum, then the sixteen are added in
// order; rows beyond float32's range are redone.  The block that finishes last adds up the losses of all rows (ignored ones hold
// 0) in one fixed order.
template <typename T>
__global__ void __launch_bounds__(512, 2) ce_sum_kernel(const CeSumArgs g) {
    __shared__ float sh[16][33];
    __shared__ double sh_d[16];
    __shared__ unsigned far;
    __shared__ bool last;
    pdl_launch_dependents();
    pdl_wait();
    const int r = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t j0 = (int64_t)blockIdx.x * 32, j = j0 + r, n = *g.rows.count;
    if (j0 < n) {
        float a = 0.0f;
        if (j < n) {
#pragma unroll 8
            for (int p = grp; p < g.nparts; p += 16) a += g.partial[(int64_t)p * g.ld_partial + j];
        }
        sh[grp][r] = a;
        __syncthreads();
        if (grp == 0) {
            float s = 0.0f;
            bool lost = false;
            if (j < n) {
#pragma unroll
                for (int k = 0; k < 16; ++k) s += sh[k][r];
                // d != 0: the others together are at least as likely as the target, or the row is redone: a small loss would come out of
                // terms that float32 no longer holds, and of a difference (not-a-number is the answer already)
                const float d = g.rows.dist[j], own = expf(-d);
                const float l = d == 0.0f ? log1pf(s) : s < 1.0f && d < 85.0f ? log1pf(s * expf(d)) : logf(s + own) + d;
                lost = s >= S_LIMIT || (d != 0.0f && (s < g.least || s < own));
                const int32_t row = g.rows.idx[j];
                g.s[j] = s;
                g.loss_rows[row] = l;
                if (g.loss_rows2) g.loss_rows2[row] = l;
                g.lse[row] = g.rows.lt[j] + l;
            }
            const unsigned f = __ballot_sync(0xffffffffu, lost);
            if (r == 0) far = f;
        }
        __syncthreads();
        for (unsigned f = far; f;) {
            ce_far_rows<T>(g, j0, f);
            for (int k = 0; k < FAR; ++k) f &= f - 1;
        }
    }
    if (!g.loss) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(g.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double a = 0.0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < g.rows.T; i += 512) a += (double)__ldcg(g.loss_rows + i);
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (r == 0) sh_d[grp] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        a = 0.0;
        for (int k = 0; k < 16; ++k) a += sh_d[k];
        *g.loss = (float)(g.mean ? a / (double)n : a);
    }
}

// x's gradient from the slots: their sum, finished with s and the target's row (noise: voc.w null and s given), written to the
// rows' own places; zeros at ignored rows.
// A block takes ROWS rows of one column tile, a thread four columns of every fourth row; what concerns a row is worked out once, by
// one thread.
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&f)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(float *p, const float (&f)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]); }
template <typename T, typename O, int ROWS>
__global__ void __launch_bounds__(CE_TILE, ROWS == 16 ? 4 : 2) ce_dx_kernel(O *__restrict__ dx, float *__restrict__ slots, const int2 *__restrict__ parts,
                                                       const int32_t *__restrict__ map, const float *__restrict__ s, const float *__restrict__ dist,
                                                       const int32_t *__restrict__ tcol, Vocab voc, int64_t T_rows, int64_t R, int tile_rows, int tiles_n) {
    __shared__ const float *sh_at[ROWS];
    __shared__ int sh_parts[ROWS];
    __shared__ uint32_t sh_hash[ROWS];             // noise word position of the target's row, column 0
    __shared__ float sh_s[ROWS], sh_inv[ROWS];  // v -> (v - s w_t) / (s + exp(-d))
    __shared__ int64_t sh_step;
    pdl_launch_dependents();
    pdl_wait();
    const int nt = (int)(blockIdx.x % (unsigned)tiles_n);
    const int64_t i0 = (int64_t)(blockIdx.x / (unsigned)tiles_n) * ROWS;
    if (threadIdx.x < ROWS) {
        const int64_t i = i0 + threadIdx.x;
        const int64_t j = i < T_rows ? map[i] : -1;
        int n = 0;
        float sj = 0.0f, inv = 1.0f;
        if (j >= 0) {
            const SlotRow o(slots, parts, tiles_n, tile_rows, j, nt);
            sh_at[threadIdx.x] = o.first;
            sh_step = o.step;                         // the same for every row
            n = o.n;
            if (s) {
                sj = s[j];
                const int32_t t = tcol[j];
                if (sj < 0.0f) {                      // the row was finished by ce_far_rows
                    n = 1;
                    sj = 0.0f;
                } else {
                    inv = t >= 0 ? 1.0f / (expf(-dist[j]) + sj) : NAN;
                }
                sh_hash[threadIdx.x] = sq5_lin_rows(voc.seed, voc.row0 + (uint32_t)t, 0u).base;
            }
        }
        sh_s[threadIdx.x] = sj;
        sh_inv[threadIdx.x] = inv;
        sh_parts[threadIdx.x] = n;
    }
    __syncthreads();
    const int cl = (threadIdx.x & 63) * 4;
    const int64_t c = (int64_t)nt * CE_TILE + cl;
    if (c >= R) return;
    const bool vec = R % 4 == 0 && (reinterpret_cast<uintptr_t>(dx) & (4 * sizeof(O) - 1)) == 0;
    float4 v[ROWS / 4];
    int most = 0;
#pragma unroll
    for (int q = 0; q < ROWS / 4; ++q) {
        const int k = (threadIdx.x >> 6) + 4 * q;
        v[q] = sh_parts[k] ? *reinterpret_cast<const float4 *>(sh_at[k] + cl) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        most = sh_parts[k] > most ? sh_parts[k] : most;
    }
#pragma unroll(ROWS == 4 ? 8 : 1)
    for (int g = 1; g < most; ++g) {
        const int64_t off = g * sh_step + cl;
#pragma unroll
        for (int q = 0; q < ROWS / 4; ++q) {
            const int k = (threadIdx.x >> 6) + 4 * q;
            if (g < sh_parts[k]) {
                const float4 u = *reinterpret_cast<const float4 *>(sh_at[k] + off);
                v[q].x += u.x; v[q].y += u.y; v[q].z += u.z; v[q].w += u.w;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < ROWS / 4; ++q) {
        const int k = (threadIdx.x >> 6) + 4 * q;
        const int64_t i = i0 + k;
        if (i >= T_rows) return;
        float f[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        if (s && sh_parts[k]) {
            const float sj = sh_s[k], inv = sh_inv[k];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = to_f32<T>(from_f32<T>(sq5_to_float(sq5_tail(sh_hash[k] + (uint32_t)(c + e) * SQ5_N1))));
                f[e] = (f[e] - sj * w) * inv;
            }
        }
        O *out = dx + i * R + c;
        if (vec) store4(out, f);
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < R) out[e] = from_f32<O>(f[e]);
        }
    }
}

// dz = unit gradient times what the loss's own gradient (and the mean's 1 / count) say
__device__ __forceinline__ void store_f8(__nv_bfloat16 *p, const float (&f)[8]) { *reinterpret_cast<uint4 *>(p) = pack_f8(f); }
__device__ __forceinline__ void store_f8(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
// ignored rows stay zero whatever the factor (no row counts: 1 / 0)
__device__ __forceinline__ float scaled(float u, float g) { return u == 0.0f ? 0.0f : u * g; }
template <typename T>
__global__ void __launch_bounds__(256) ce_scale_kernel(T *__restrict__ dz, const float *__restrict__ unit, const float *__restrict__ dloss,
                                                       const float *__restrict__ count, int64_t rows, int64_t R, int reduction) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t total = rows * R;
    const float g0 = reduction == RDB_CE_NONE ? 0.0f : reduction == RDB_CE_MEAN ? dloss[0] / *count : dloss[0];
    const bool vec = R % 8 == 0 && ((reinterpret_cast<uintptr_t>(dz) | reinterpret_cast<uintptr_t>(unit)) & 15) == 0;
    if (vec) {
        const int64_t groups = total / 8, per = R / 8;
        for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < groups; i += (int64_t)gridDim.x * blockDim.x) {
            const float g = reduction == RDB_CE_NONE ? dloss[i / per] : g0;
            float f[8];
            load_f8(f, unit + i * 8);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = scaled(f[k], g);
            store_f8(dz + i * 8, f);
        }
        return;
    }
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x)
        dz[i] = from_f32<T>(scaled(unit[i], reduction == RDB_CE_NONE ? dloss[i / R] : g0));
}

// ================================================================================================
// a few rows, loss only
// ================================================================================================
// Scoring a token or a few: the matrix is read (or hashed) once and multiplied on CUDA cores; a tile of the tensor-core path would
// be 250 rows of padding, behind four kernels that prepare it.  A warp takes FEW_ROWS vocabulary rows at a time, 32 lanes along the
// columns, the rows of x in shared memory; each lane ends up with the logits of some (vocabulary row, x row) pairs and keeps a running
// maximum and a sum relative to it.  Bound by the launches where small, by the hash (noise) or the matrix's bytes (stored) where large.
// Against the tensor-core path, on the device, us, V = 50257 but where said:
//   bf16   1 x 128  noise 33 -> 18, stored 31 -> 16     4 x 768  noise 66 -> 55, stored 40 -> 41
//          V = 128256: 1 x 4096  noise 608 -> 424, stored 221 -> 211 (5.0 TB/s)     4 x 2048  noise 401 -> 250, stored 123 -> 127
//   fp32   1 x 128  noise 53 -> 18, stored 51 -> 18     4 x 768  noise 174 -> 53, stored 182 -> 51
// Four rows of bf16 are where the two meet for a stored matrix: each value is loaded once, but converted and multiplied per row.
constexpr int FEW_T = 4;                      // rows of x at most
constexpr int FEW_ROWS = 4;                   // vocabulary rows per warp and pass
constexpr int FEW_WARPS = 8;
// blocks per SM, as many as the registers and shared memory of each form hold at once: every warp has the same share of the rows
constexpr int few_blocks(int nt, bool noise) { return noise ? 4 : nt == 1 ? 3 : 2; }

struct FewArgs {
    const void *x;
    int64_t ldx, T, R, V;
    const int64_t *target;
    Vocab voc;
    float2 *partial;                          // (maximum, sum relative to it) per block and row of x
    int64_t ignore;
    int use_ignore, mean;
    float *lse, *loss_rows, *loss_rows2, *count, *loss;
};

// rows of x in shared memory start at 16 bytes
__host__ __device__ __forceinline__ int few_stride(int64_t R) { return (int)((R + 3) / 4 * 4); }

template <typename T, int NT, bool NOISE>
__global__ void __launch_bounds__(FEW_WARPS * 32, few_blocks(NT, NOISE)) ce_few_kernel(const FewArgs a) {
    extern __shared__ __align__(16) float xs[];   // [NT][RS]
    __shared__ float2 sh[FEW_WARPS][NT];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int R = (int)a.R, RS = few_stride(R);
    for (int t = 0; t < NT; ++t)
        for (int c = threadIdx.x; c < R; c += FEW_WARPS * 32)
            xs[t * RS + c] = t < a.T ? to_f32<T>(reinterpret_cast<const T *>(a.x)[t * a.ldx + c]) : 0.0f;
    __syncthreads();
    // lane i takes the sum of pair i of (vocabulary row, x row): row i / NT, x row i % NT
    constexpr int PAIRS = FEW_ROWS * NT;
    const int my_row = (lane % PAIRS) / NT, my_t = lane % NT;
    const int64_t my_target = my_t < a.T ? a.target[my_t] : -1;
    float m = -INFINITY, s = 0.0f;
    const bool vec = !NOISE && rows_aligned<T>(a.voc.w, a.voc.ldw);
    constexpr int W = 16 / sizeof(T);         // elements of a 16-byte load
    const int64_t step = (int64_t)gridDim.x * FEW_WARPS * FEW_ROWS;
    for (int64_t v0 = ((int64_t)blockIdx.x * FEW_WARPS + warp) * FEW_ROWS; v0 < a.V; v0 += step) {
        float acc[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) acc[i] = 0.0f;
        int c = 0;                            // columns done
        if (NOISE) {
            uint32_t h[FEW_ROWS];
#pragma unroll
            for (int r = 0; r < FEW_ROWS; ++r) h[r] = sq5_lin_rows(a.voc.seed, a.voc.row0 + (uint32_t)(v0 + r), (uint32_t)lane).base;
#pragma unroll 2
            for (c = lane; c < R; c += 32) {
                float w[FEW_ROWS];
#pragma unroll
                for (int r = 0; r < FEW_ROWS; ++r) {
                    w[r] = to_f32<T>(from_f32<T>(sq5_to_float(sq5_tail(h[r]))));
                    h[r] += 32u * SQ5_N1;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float x = xs[t * RS + c];
#pragma unroll
                    for (int r = 0; r < FEW_ROWS; ++r) acc[r * NT + t] = fmaf(x, w[r], acc[r * NT + t]);
                }
            }
        } else {
            const T *row[FEW_ROWS];
#pragma unroll
            for (int r = 0; r < FEW_ROWS; ++r) row[r] = reinterpret_cast<const T *>(a.voc.w) + (v0 + r < a.V ? v0 + r : a.V - 1) * a.voc.ldw;
            const int whole = vec ? R / W * W : 0;
#pragma unroll 2
            for (c = lane * W; c < whole; c += 32 * W) {
                uint4 u[FEW_ROWS];
#pragma unroll
                for (int r = 0; r < FEW_ROWS; ++r) u[r] = __ldg(reinterpret_cast<const uint4 *>(row[r] + c));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int e = 0; e < W; e += 4) {
                        const float4 q = *reinterpret_cast<const float4 *>(xs + t * RS + c + e);
                        const float x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int r = 0; r < FEW_ROWS; ++r)
                                acc[r * NT + t] = fmaf(x[k], to_f32<T>(reinterpret_cast<const T *>(&u[r])[e + k]), acc[r * NT + t]);
                    }
                }
            }
            for (c = whole + lane; c < R; c += 32) {
#pragma unroll
                for (int r = 0; r < FEW_ROWS; ++r) {
                    const float w = to_f32<T>(row[r][c]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[r * NT + t] = fmaf(xs[t * RS + c], w, acc[r * NT + t]);
                }
            }
        }
        const float l = warp_sums(acc, lane);
        const int64_t v = v0 + my_row;
        if (lane < PAIRS && v < a.V && v != my_target) online(m, s, l);
    }
    // lanes of the same x row, then the warps
#pragma unroll
    for (int o = NT; o < 32; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        online_join(m, s, m2, s2);
    }
    if (lane < NT) sh[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < NT) {
        float2 r = sh[0][threadIdx.x];
        for (int k = 1; k < FEW_WARPS; ++k) online_join(r.x, r.y, sh[k][threadIdx.x].x, sh[k][threadIdx.x].y);
        a.partial[(int64_t)blockIdx.x * NT + threadIdx.x] = r;
    }
}

// one block: a warp per row joins the blocks' sums and computes the target's logit
template <typename T, int NT>
__global__ void __launch_bounds__(FEW_T * 32) ce_few_finish_kernel(const FewArgs a, int blocks) {
    __shared__ float sh_loss[FEW_T];
    __shared__ int sh_kept[FEW_T];
    pdl_wait();
    // not before: blocks of a next call that come while this call's still run would fill some SMs twice over, and the shares
    // are fixed (1 row of 4096, V = 128256, noise, calls in a row: 790 us, against 465 us for one alone)
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, t = threadIdx.x >> 5;
    if (t < a.T) {
        float m = -INFINITY, s = 0.0f, lt = 0.0f;
        for (int b = lane; b < blocks; b += 32) {
            const float2 p = a.partial[(int64_t)b * NT + t];
            online_join(m, s, p.x, p.y);
        }
        const int64_t target = a.target[t];
        const bool known = target >= 0 && target < a.V;
        const T *x = reinterpret_cast<const T *>(a.x) + t * a.ldx;
        if (known)
            for (int64_t c = lane; c < a.R; c += 32) lt = fmaf(to_f32<T>(x[c]), vocab_at<T>(a.voc, target, c), lt);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
            online_join(m, s, m2, s2);
            lt += __shfl_xor_sync(0xffffffffu, lt, o);
        }
        const bool kept = !(a.use_ignore && target == a.ignore);
        // relative to the target's logit while that holds, as everywhere else
        const float up = m - lt;
        float loss = loss_above(up, s);
        if (!known) loss = NAN;
        if (!(lt == lt) || !(m == m)) loss = NAN;
        if (!kept) loss = 0.0f;
        if (lane == 0) {
            a.loss_rows[t] = loss;
            if (a.loss_rows2) a.loss_rows2[t] = loss;
            a.lse[t] = kept ? lt + loss : 0.0f;
            sh_loss[t] = loss;
            sh_kept[t] = kept;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        int n = 0;
        for (int k = 0; k < a.T; ++k) {
            sum += sh_loss[k];
            n += sh_kept[k];
        }
        *a.count = (float)n;
        if (a.loss) *a.loss = (float)(a.mean ? sum / n : sum);
    }
}

template <typename T, int NT>
static int launch_few(const FewArgs &a, cudaStream_t st) {
    const int64_t want = cdiv64(a.V, FEW_WARPS * FEW_ROWS);
    const int64_t most = (int64_t)sm_count() * few_blocks(NT, !a.voc.w);
    const int blocks = (int)(want < most ? want : most);
    const size_t smem = (size_t)NT * few_stride(a.R) * sizeof(float);
    const int rc = a.voc.w ? launch_pdl(ce_few_kernel<T, NT, false>, dim3(blocks), FEW_WARPS * 32, smem, st, a)
                           : launch_pdl(ce_few_kernel<T, NT, true>, dim3(blocks), FEW_WARPS * 32, smem, st, a);
    if (rc) return rc;
    return launch_pdl(ce_few_finish_kernel<T, NT>, dim3(1), FEW_T * 32, 0, st, a, blocks);
}

// whether a loss without a gradient takes this way: its rows of x fit the 48 KB of shared memory that
// need no opting in, with the kernel's own few hundred bytes
static bool few_rows(int64_t T, int64_t R) { return T >= 1 && T <= FEW_T && R <= 47 * 1024 / (int64_t)sizeof(float) / (T == 1 ? 1 : FEW_T) - 4; }

// ================================================================================================
// host side
// ================================================================================================
struct CePlan {
    int parts, nterm;
    int64_t Mpad, Rp, lda;           // rows rounded to tiles; columns of one part, of all parts
    int64_t piece, npieces;          // vocabulary columns per piece (a multiple of 256), pieces
    bool stage_b;                    // the matrix goes through the workspace in bf16 parts
    int pairs, tile_rows;
    int64_t slot_rows;               // rows of 256 float32 that the parts of the x-gradient take
    bool dw_direct;
    int64_t ld_dw;
    // workspace
    size_t idx, map, count, off2, lt, dist, scale, tval, tcol, s, ticket, a, b, e, partial, slots, parts_at, dw, tail, total;
    bool slots_used;
};

constexpr size_t E_BUDGET = 512ull << 20;
constexpr size_t B_BUDGET = 256ull << 20;

static int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

static int ce_kb(const CePlan &p) { return p.nterm * (int)cdiv64(p.piece, BK); }     // k-blocks of the x-gradient's product

// Rows per tile.  float32: 256 (the registers hold one sub-tile).  bf16: 512-row tiles are the faster ones where rows fill them (8192
// rows; 4000 of R = 1024, V = 50257, loss and gradient: 683 against 724 us), by about a tenth: 256-row tiles win when they round the
// rows up to a tenth less (600 rows: 183 against 214; 2100: 410 against 454; 1200: even), and for short contractions of few rows, where
// the exponentials bound the logits and twice the tiles spread better (V = 32003, us, loss and gradient: R = 200 512 rows 66 against 69, 1600 rows
// 105 against 113; R = 512 82 against 87, 146 against 158, 2048 rows 159 against 160; R = 640 95 against 98, 179 against 189, but 2048 rows 196 against
// 194; R = 200 4000 rows 177 against 173).
static int ce_tile_rows(int64_t T, int64_t R, int dtype) {
    if (dtype == RDB_F32) return CE_TILE;
    const int64_t r256 = round_up(T, CE_TILE), r512 = round_up(T, 2 * CE_TILE);
    return r256 * 11 < r512 * 10 || (R <= 512 && T <= 2048) ? CE_TILE : 2 * CE_TILE;
}

// op 0: loss; 1: loss and unit gradient of x (noise); 2: gradients of a stored matrix
static CePlan ce_plan(int op, int64_t T, int64_t R, int64_t V, int dtype, const void *w, int64_t ldw, const void *dw, int want_dx, int want_dw) {
    CePlan p{};
    if (op == 0 && few_rows(T, R)) {          // partial sums of ce_few_kernel only
        p.total = (size_t)sm_count() * few_blocks(1, true) * FEW_T * sizeof(float2);
        return p;
    }
    p.parts = dtype == RDB_F32 ? 3 : 1;
    p.nterm = dtype == RDB_F32 ? 6 : 1;
    p.tile_rows = ce_tile_rows(T, R, dtype);
    p.Mpad = round_up(T, p.tile_rows);
    p.Rp = round_up(R, p.parts == 3 ? 64 : 8);
    p.lda = p.Rp * p.parts;
    p.pairs = max_resident_pairs();
    // a stored bf16 matrix whose rows start on 16-byte boundaries is read where it is
    p.stage_b = !(w && dtype == RDB_BF16 && (ldw % 8) == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0);
    const int64_t vtiles = cdiv64(V, CE_TILE);
    int64_t most = vtiles;
    if (op != 0) {
        const int64_t m = (int64_t)(E_BUDGET / ((size_t)p.Mpad * p.parts * 2 * CE_TILE + 1));
        most = m < most ? m : most;
    }
    if (p.stage_b) {
        const int64_t m = (int64_t)(B_BUDGET / ((size_t)p.lda * 2 * CE_TILE));
        most = m < most ? m : most;
    }
    if (most < 1) most = 1;
    p.npieces = cdiv64(vtiles, most);
    const int64_t per = cdiv64(vtiles, p.npieces);
    p.npieces = cdiv64(vtiles, per);
    p.piece = per * CE_TILE;
    p.slot_rows = (int64_t)Cut(T, R, ce_kb(p), p.pairs, p.tile_rows).slots(p.pairs) * p.tile_rows;
    const size_t es = dtype_size(dtype);
    p.dw_direct = dw && (reinterpret_cast<uintptr_t>(dw) & 15) == 0 && (R * es) % 16 == 0;
    p.ld_dw = round_up(R, 8);
    size_t o = 0;
    auto take = [&](size_t bytes) { const size_t at = o; o += align_up(bytes, 1024); return at; };
    p.idx = take((size_t)p.Mpad * 4);
    p.map = take((size_t)T * 4);
    p.count = take(16);
    p.off2 = take((size_t)p.Mpad * 4);
    p.tcol = take((size_t)p.Mpad * 4);
    p.lt = take((size_t)p.Mpad * 4);
    p.dist = take((size_t)p.Mpad * 4);
    p.s = take((size_t)p.Mpad * 4);
    p.ticket = take(16);
    p.scale = take(op == 2 ? (size_t)p.Mpad * 4 : 0);
    p.tval = take(op == 2 ? (size_t)p.Mpad * 4 : 0);
    p.a = take((size_t)p.Mpad * p.lda * 2);
    p.b = take(p.stage_b ? (size_t)p.piece * p.lda * 2 : 0);
    p.e = take(op != 0 ? (size_t)p.Mpad * p.piece * p.parts * 2 : 0);
    p.partial = take(op != 2 ? (size_t)p.npieces * (p.piece / CE_TILE) * 2 * p.Mpad * 4 : 0);
    p.slots_used = op == 1 || (op == 2 && want_dx);
    p.slots = take(p.slots_used ? (size_t)p.slot_rows * CE_TILE * 4 : 0);
    p.parts_at = take(p.slots_used ? (size_t)(p.Mpad / p.tile_rows) * cdiv64(cdiv64(R, CE_TILE), 8) * 8 : 0);
    p.dw = take(op == 2 && want_dw && !p.dw_direct ? (size_t)p.piece * p.ld_dw * es : 0);
    p.tail = take(op == 2 && want_dw ? (size_t)p.pairs * p.tile_rows * CE_TILE * 4 : 0);
    p.total = o;
    return p;
}

static void ce_terms(CeArgs *a, int nterm, int64_t a_cols, int64_t b_cols) {
    a->nterm = nterm;
    static const int pa[6] = {0, 1, 2, 0, 1, 0}, pb[6] = {2, 1, 0, 1, 0, 0};    // smallest first
    for (int i = 0; i < nterm; ++i) {
        a->a_off[i] = nterm == 1 ? 0 : (int)(pa[i] * a_cols);
        a->b_off[i] = nterm == 1 ? 0 : (int)(pb[i] * b_cols);
    }
}

template <int A_MN, int B_MN, int EPI, int PARTS, int MT>
static int launch_pair(const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &td, const CUtensorMap &ts, const CeArgs &args,
                       int64_t max_items, int pairs, cudaStream_t st) {
    auto kern = ce_pair_kernel<A_MN, B_MN, EPI, PARTS, MT>;
    static std::atomic<uint64_t> prepared{0};          // devices on which the kernel may use its shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64 || !((prepared.load() >> dev) & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, CeCfg<MT>::SMEM);
        if (e != cudaSuccess) return (int)e;
        if (dev < 64) prepared.fetch_or(1ull << dev);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(CE_THREADS);
    cfg.dynamicSmemBytes = CeCfg<MT>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const int64_t n = max_items < pairs ? max_items : pairs;
    cfg.gridDim = dim3((unsigned)(2 * (n < 1 ? 1 : n)));
    e = cudaLaunchKernelEx(&cfg, kern, ta, tb, td, ts, args);
    if (e != cudaSuccess) return (int)e;
    return launch_status();
}

struct CeCall {
    CePlan p;
    uint8_t *ws;
    const void *x;
    int64_t ldx, T, R, V;
    Vocab voc;
    const int64_t *target;
    int dtype;
    int32_t *status;
    cudaStream_t st;
    template <typename P> P *at(size_t off) const { return reinterpret_cast<P *>(ws + off); }
};

static int ce_find_rows(const CeCall &c, int64_t ignore, int use_ignore, float *zero_a, float *zero_b, float *zero_c, float *count_f) {
    return launch_pdl(ce_rows_kernel, dim3(1), 1024, 0, c.st, c.target, c.T, ignore, use_ignore, c.at<int32_t>(c.p.idx), c.at<int32_t>(c.p.map),
                      c.at<int32_t>(c.p.count), zero_a, zero_b, zero_c, count_f, c.at<uint32_t>(c.p.ticket), c.p.slots_used ? c.at<int2>(c.p.parts_at) : (int2 *)nullptr, c.R, ce_kb(c.p),
                      c.p.pairs, c.p.tile_rows);
}

// Mean of the largest of n standard normal values, by its limiting (Gumbel) distribution; its spread is 1.28 / sqrt(2 ln n).
static float largest_of(int64_t n) {
    const double a = sqrt(2.0 * log((double)n));
    return n < 16 ? (float)a : (float)(a + (0.5772 - 0.5 * (log(log((double)n)) + log(4.0 * 3.14159265))) / a);
}

static CeRowArgs ce_row_args(const CeCall &c) {
    CeRowArgs a{};
    a.x = c.x; a.ldx = c.ldx; a.T = c.T; a.R = c.R; a.V = c.V;
    a.target = c.target;
    a.idx = c.at<int32_t>(c.p.idx);
    a.count = c.at<int32_t>(c.p.count);
    a.a = c.at<__nv_bfloat16>(c.p.a);
    a.lda = c.p.lda; a.part_cols = c.p.Rp;
    a.off2 = c.at<float>(c.p.off2);
    a.lt = c.at<float>(c.p.lt);
    a.dist = c.at<float>(c.p.dist);
    a.spread = largest_of(c.V);
    a.scale = c.at<float>(c.p.scale);
    a.tval = c.at<float>(c.p.tval);
    a.tcol = c.at<int32_t>(c.p.tcol);
    a.tile_rows = c.p.tile_rows;
    return a;
}

static int ce_gather(const CeCall &c, const CeRowArgs &a) {
    const dim3 grid((unsigned)(c.p.Mpad / 8));
    if (c.dtype == RDB_F32) return launch_pdl(ce_gather_kernel<float, 3>, grid, 256, 0, c.st, a, c.voc);
    return launch_pdl(ce_gather_kernel<__nv_bfloat16, 1>, grid, 256, 0, c.st, a, c.voc);
}

// The matrix's rows [v0, v0 + n) as a bf16 operand: where it starts and its pitch.
static int ce_stage(const CeCall &c, int64_t v0, int64_t n, const void **base, int64_t *ld) {
    if (!c.p.stage_b) {
        *base = reinterpret_cast<const __nv_bfloat16 *>(c.voc.w) + v0 * c.voc.ldw;
        *ld = c.voc.ldw;
        return RDB_OK;
    }
    __nv_bfloat16 *b = c.at<__nv_bfloat16>(c.p.b);
    *base = b;
    *ld = c.p.lda;
    if (!c.voc.w && c.dtype == RDB_BF16)
        return rdb_noise(b, RDB_BF16, n, c.R, c.p.lda, (int64_t)c.voc.row0 + v0, 0, c.voc.seed, c.st);
    const int64_t want = cdiv64(n * c.p.Rp / 8, 256);
    const dim3 grid((unsigned)(want < 148 * 8 ? (want < 1 ? 1 : want) : 148 * 8));
    if (c.dtype == RDB_F32) return launch_pdl(ce_split_kernel<float, 3>, grid, 256, 0, c.st, b, c.p.lda, c.p.Rp, n, c.R, v0, c.voc);
    return launch_pdl(ce_split_kernel<__nv_bfloat16, 1>, grid, 256, 0, c.st, b, c.p.lda, c.p.Rp, n, c.R, v0, c.voc);
}

// logits of one piece through the epilogue EPI
template <int EPI>
static int ce_logits(const CeCall &c, const void *b, int64_t ldb, int64_t v0, int64_t n, int64_t piece_index) {
    const CePlan &p = c.p;
    const int64_t width = p.parts == 1 ? c.R : p.lda;              // columns beyond read as zero
    CUtensorMap ta, tb, td;
    int rc = make_tmap(&ta, c.at<void>(p.a), width, p.Mpad, p.lda, BK, BM);
    if (rc) return rc;
    rc = make_tmap(&tb, b, width, n, ldb, BK, BM);
    if (rc) return rc;
    td = ta;
    CeArgs a{};
    if (EPI != EPI_SUM) {
        rc = make_tmap(&td, c.at<void>(p.e), p.piece * p.parts, p.Mpad, p.piece * p.parts, 32, 32, false, CU_TENSOR_MAP_SWIZZLE_64B);
        if (rc) return rc;
    }
    a.count = c.at<int32_t>(p.count);
    a.m_counted = 1;
    a.N = p.piece;                    // columns past the vocabulary's end come out as zeros
    if (EPI == EPI_SUM) a.N = n;
    a.kbs = (int)cdiv64(p.parts == 1 ? c.R : p.Rp, BK);
    ce_terms(&a, p.nterm, p.Rp, p.Rp);
    a.m_fast = 1;
    a.off2 = c.at<float>(p.off2);
    a.scale = c.at<float>(p.scale);
    a.tval = c.at<float>(p.tval);
    a.tcol = c.at<int32_t>(p.tcol);
    a.v0 = (int32_t)v0;
    a.ncols = (int32_t)n;
    a.partial = c.at<float>(p.partial) + piece_index * (p.piece / CE_TILE) * 2 * p.Mpad;
    a.ld_partial = p.Mpad;
    a.part_cols = (int)p.piece;
    a.status = c.status;
    const int64_t items = (p.Mpad / p.tile_rows) * cdiv64(a.N, CE_TILE);
    if (p.parts == 3) return launch_pair<0, 0, EPI, 3, 1>(ta, tb, td, td, a, items, p.pairs, c.st);
    if (p.tile_rows == CE_TILE) return launch_pair<0, 0, EPI, 1, 1>(ta, tb, td, td, a, items, p.pairs, c.st);
    return launch_pair<0, 0, EPI, 1, 2>(ta, tb, td, td, a, items, p.pairs, c.st);
}

// slots (+)= E W_piece
static int ce_accumulate(const CeCall &c, const void *b, int64_t ldb, int64_t n, bool add) {
    const CePlan &p = c.p;
    CUtensorMap ta, tb, td;
    int rc = make_tmap(&ta, c.at<void>(p.e), p.piece * p.parts, p.Mpad, p.piece * p.parts, BK, BM);
    if (rc) return rc;
    rc = make_tmap(&tb, b, p.parts == 1 ? c.R : p.lda, n, ldb, 64, BK);
    if (rc) return rc;
    rc = make_tmap(&td, c.at<void>(p.slots), CE_TILE, p.slot_rows, CE_TILE, 32, 32, true);
    if (rc) return rc;
    CeArgs a{};
    a.count = c.at<int32_t>(p.count);
    a.m_counted = 1;
    a.N = c.R;
    a.kbs = (int)cdiv64(p.piece, BK);
    ce_terms(&a, p.nterm, p.piece, p.Rp);
    a.m_fast = 0;
    a.accumulate = add ? 1 : 0;
    a.status = c.status;
    if (p.parts == 3) return launch_pair<0, 1, EPI_SLOT, 3, 1>(ta, tb, td, td, a, p.pairs, p.pairs, c.st);
    if (p.tile_rows == CE_TILE) return launch_pair<0, 1, EPI_SLOT, 1, 1>(ta, tb, td, td, a, p.pairs, p.pairs, c.st);
    return launch_pair<0, 1, EPI_SLOT, 1, 2>(ta, tb, td, td, a, p.pairs, p.pairs, c.st);
}

// dW rows [v0, v0 + n) = P^T x
static int ce_dw(const CeCall &c, void *dw, int64_t v0, int64_t n) {
    const CePlan &p = c.p;
    const size_t es = dtype_size(c.dtype);
    const int64_t ldd = p.dw_direct ? c.R : p.ld_dw;
    void *out = p.dw_direct ? static_cast<void *>(static_cast<uint8_t *>(dw) + (size_t)v0 * c.R * es) : c.at<void>(p.dw);
    CUtensorMap ta, tb, td;
    int rc = make_tmap(&ta, c.at<void>(p.e), p.piece * p.parts, p.Mpad, p.piece * p.parts, 64, BK);
    if (rc) return rc;
    rc = make_tmap(&tb, c.at<void>(p.a), p.parts == 1 ? c.R : p.lda, p.Mpad, p.lda, 64, BK);
    if (rc) return rc;
    rc = c.dtype == RDB_F32 ? make_tmap(&td, out, c.R, n, ldd, 32, 32, true) : make_tmap(&td, out, c.R, n, ldd, 32, 32, false, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
    CeArgs a{};
    a.count = c.at<int32_t>(p.count);
    a.k_counted = 1;
    a.M = n;
    a.N = c.R;
    ce_terms(&a, p.nterm, p.piece, p.Rp);
    a.m_fast = 0;
    a.status = c.status;
    // Tiles that do not fill the last round of pairs are cut along the contraction when two or more pairs can share each; their
    // parts go through slots of their own.
    const int tile_rows = p.tile_rows;
    const int64_t tiles = cdiv64(n, tile_rows) * cdiv64(c.R, CE_TILE);
    const int left = (int)(tiles % p.pairs);
    const int64_t kb = a.nterm * cdiv64(c.T, BK);
    a.tail_parts = 1;
    if (left > 0 && p.pairs / left >= 2 && kb >= 8) {
        int64_t parts = p.pairs / left;
        if (parts > kb / 4) parts = kb / 4;
        a.tail = left;
        a.tail_parts = (int)parts;
    }
    CUtensorMap ts = td;
    float *tail = c.at<float>(p.tail);
    if (a.tail && (rc = make_tmap(&ts, tail, CE_TILE, (int64_t)p.pairs * tile_rows, CE_TILE, 32, 32, true))) return rc;
    const int64_t items = tiles - a.tail + (int64_t)a.tail * a.tail_parts;
    rc = c.dtype == RDB_F32 ? launch_pair<1, 1, EPI_F32, 3, 1>(ta, tb, td, ts, a, items, p.pairs, c.st)
         : tile_rows == CE_TILE ? launch_pair<1, 1, EPI_BF16, 1, 1>(ta, tb, td, ts, a, items, p.pairs, c.st)
                                : launch_pair<1, 1, EPI_BF16, 1, 2>(ta, tb, td, ts, a, items, p.pairs, c.st);
    if (rc) return rc;
    uint8_t *mine = static_cast<uint8_t *>(dw) + (size_t)v0 * c.R * es;
    if (!p.dw_direct && tiles > a.tail) {
        // whole tiles came to the padded copy: as many rows as have one
        const int64_t rows = round_up(tiles - a.tail, cdiv64(c.R, CE_TILE)) / cdiv64(c.R, CE_TILE) * tile_rows;
        const int64_t m = rows < n ? rows : n;
        const dim3 grid((unsigned)cdiv64(m, 4));
        rc = c.dtype == RDB_F32 ? launch_pdl(ce_copy_kernel<float>, grid, 256, 0, c.st, (float *)mine, (const float *)out, m, c.R, ldd)
                                : launch_pdl(ce_copy_kernel<__nv_bfloat16>, grid, 256, 0, c.st, (__nv_bfloat16 *)mine, (const __nv_bfloat16 *)out, m, c.R, ldd);
        if (rc) return rc;
    }
    if (a.tail) {
        const dim3 grid((unsigned)(a.tail * (tile_rows / 4)));
        const int first = (int)(tiles - a.tail);
        rc = c.dtype == RDB_F32 ? launch_pdl(ce_tail_kernel<float>, grid, 256, 0, c.st, (float *)mine, c.R, (const float *)tail, n, c.R, first, a.tail_parts, tile_rows)
                                : launch_pdl(ce_tail_kernel<__nv_bfloat16>, grid, 256, 0, c.st, (__nv_bfloat16 *)mine, c.R, (const float *)tail, n, c.R, first, a.tail_parts, tile_rows);
    }
    return rc;
}

static int ce_finish_dx(const CeCall &c, void *dx, bool unit) {
    const CePlan &p = c.p;
    const int tiles_n = (int)cdiv64(c.R, CE_TILE);
    const float *s = unit ? c.at<float>(p.s) : nullptr, *dist = c.at<float>(p.dist);
    const int32_t *map = c.at<int32_t>(p.map), *tcol = c.at<int32_t>(p.tcol);
    const int2 *parts = c.at<int2>(p.parts_at);
    float *slots = c.at<float>(p.slots);
    // few rows have many parts each and are bound by latency: four rows per block then (1531 rows of 200: 12 against 24 us)
    const int rows = cdiv64(c.T, 16) * tiles_n >= 4 * 148 ? 16 : 4;
    const dim3 grid((unsigned)(cdiv64(c.T, rows) * tiles_n));
    auto go = [&](auto kern, auto *out) {
        return launch_pdl(kern, grid, CE_TILE, 0, c.st, out, slots, parts, map, s, dist, tcol, c.voc, c.T, c.R, p.tile_rows, tiles_n);
    };
    using H = __nv_bfloat16;
    if (c.dtype == RDB_F32) return rows == 16 ? go(ce_dx_kernel<float, float, 16>, (float *)dx) : go(ce_dx_kernel<float, float, 4>, (float *)dx);
    if (unit) return rows == 16 ? go(ce_dx_kernel<H, float, 16>, (float *)dx) : go(ce_dx_kernel<H, float, 4>, (float *)dx);
    return rows == 16 ? go(ce_dx_kernel<H, H, 16>, (H *)dx) : go(ce_dx_kernel<H, H, 4>, (H *)dx);
}

static int ce_check(int64_t T, int64_t R, int64_t V, int64_t ldx, const void *w, int64_t ldw, int dtype, int reduction) {
    if (T < 0 || R < 1 || V < 1 || ldx < R || (w && ldw < R)) return RDB_ERR_SHAPE;
    if (dtype != RDB_F32 && dtype != RDB_BF16) return RDB_ERR_DTYPE;
    if (reduction != RDB_CE_NONE && reduction != RDB_CE_MEAN && reduction != RDB_CE_SUM) return RDB_ERR_UNSUPPORTED;
    // coordinates of the tiled copies and counts of tiles and k-blocks are 32-bit
    if (T > (1LL << 28) || V > (1LL << 30) || R > (1LL << 20) || (double)T * (double)R > (double)(1LL << 36) || (double)T * (double)V > (double)(1LL << 45))
        return RDB_ERR_TOO_LARGE;
    if (max_resident_pairs() < 8) return RDB_ERR_UNSUPPORTED;      // the x-gradient's groups have up to eight pairs
    return RDB_OK;
}

}  // namespace rdb

using namespace rdb;

extern "C" size_t rdb_ce_workspace_bytes(int op, int64_t T, int64_t R, int64_t V, int dtype, const void *w, int64_t ldw) {
    if (op < RDB_CE_LOSS || op > RDB_CE_GRADS || ce_check(T, R, V, R, w, ldw, dtype, RDB_CE_SUM) != RDB_OK) return 1024;
    return ce_plan(op, T, R, V, dtype, w, ldw, nullptr, 1, 1).total;
}

extern "C" int rdb_ce_fwd(float *loss, float *aux, float *dx_unit, const void *x, int64_t ldx, const void *w, int64_t ldw, const int64_t *target,
                          void *workspace, size_t workspace_bytes, int64_t T, int64_t R, int64_t V, int64_t row0, uint32_t seed,
                          int64_t ignore_index, int use_ignore, int dtype, int reduction, int32_t *status, void *stream) {
    int rc = ce_check(T, R, V, ldx, w, ldw, dtype, reduction);
    if (rc) return rc;
    if (dx_unit && w) return RDB_ERR_UNSUPPORTED;        // a stored matrix takes its gradients in rdb_ce_bwd
    if (!aux || (!loss && (T > 0 || reduction != RDB_CE_NONE))) return RDB_ERR_NULL;
    if (T > 0 && (!x || !target)) return RDB_ERR_NULL;
    const size_t es = dtype_size(dtype);
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & (es - 1)) || ((reinterpret_cast<uintptr_t>(dx_unit) | reinterpret_cast<uintptr_t>(loss) | reinterpret_cast<uintptr_t>(aux)) & 3) ||
        (reinterpret_cast<uintptr_t>(target) & 7))
        return RDB_ERR_ALIGN;
    CeCall c{};
    c.p = ce_plan(dx_unit ? 1 : 0, T, R, V, dtype, w, ldw, nullptr, 1, 0);
    if (!workspace || workspace_bytes < c.p.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return RDB_ERR_WORKSPACE;
    c.ws = reinterpret_cast<uint8_t *>(workspace);
    c.x = x; c.ldx = ldx; c.T = T; c.R = R; c.V = V;
    c.voc = Vocab{w, ldw, seed, (uint32_t)row0};
    c.target = target;
    c.dtype = dtype;
    c.status = status;
    c.st = (cudaStream_t)stream;
    float *lse = aux, *rows = aux + T, *count_f = aux + 2 * T;
    float *rows2 = reduction == RDB_CE_NONE ? loss : nullptr;       // the caller's own copy of the rows' losses
    if (!dx_unit && few_rows(T, R)) {
        FewArgs f{};
        f.x = x; f.ldx = ldx; f.T = T; f.R = R; f.V = V;
        f.target = target;
        f.voc = c.voc;
        f.partial = c.at<float2>(0);
        f.ignore = ignore_index;
        f.use_ignore = use_ignore;
        f.mean = reduction == RDB_CE_MEAN ? 1 : 0;
        f.lse = lse; f.loss_rows = rows; f.loss_rows2 = rows2; f.count = count_f;
        f.loss = reduction == RDB_CE_NONE ? nullptr : loss;
        if (dtype == RDB_F32) return T == 1 ? launch_few<float, 1>(f, c.st) : launch_few<float, FEW_T>(f, c.st);
        return T == 1 ? launch_few<__nv_bfloat16, 1>(f, c.st) : launch_few<__nv_bfloat16, FEW_T>(f, c.st);
    }
    if ((rc = ce_find_rows(c, ignore_index, use_ignore, lse, rows, rows2, count_f))) return rc;
    if (T > 0) {
        const CeRowArgs ra = ce_row_args(c);
        if ((rc = ce_gather(c, ra))) return rc;
        for (int64_t i = 0; i < c.p.npieces; ++i) {
            const int64_t v0 = i * c.p.piece, n = V - v0 < c.p.piece ? V - v0 : c.p.piece;
            const void *b;
            int64_t ldb;
            if ((rc = ce_stage(c, v0, n, &b, &ldb))) return rc;
            if (dx_unit) {
                if ((rc = ce_logits<EPI_EXP>(c, b, ldb, v0, n, i))) return rc;
                if ((rc = ce_accumulate(c, b, ldb, n, i > 0))) return rc;
            } else if ((rc = ce_logits<EPI_SUM>(c, b, ldb, v0, n, i))) return rc;
        }
    }
    // row sums: a full piece leaves two per column tile; without the gradient the last piece has only the tiles that exist
    const int64_t last = V - (c.p.npieces - 1) * c.p.piece;
    CeSumArgs g{};
    g.rows = ce_row_args(c);
    g.voc = c.voc;
    g.partial = c.at<float>(c.p.partial);
    g.ld_partial = c.p.Mpad;
    g.nparts = (int)((c.p.npieces - 1) * (c.p.piece / CE_TILE) * 2 + (dx_unit ? c.p.piece / CE_TILE : cdiv64(last, CE_TILE)) * 2);
    g.s = c.at<float>(c.p.s);
    g.lse = lse;
    g.loss_rows = rows;
    g.loss_rows2 = rows2;
    g.slots = dx_unit ? c.at<float>(c.p.slots) : nullptr;
    g.parts = c.at<int2>(c.p.parts_at);
    g.loss = reduction == RDB_CE_NONE ? nullptr : loss;
    g.mean = reduction == RDB_CE_MEAN ? 1 : 0;
    g.least = (float)V * TERM_LEAST;
    g.ticket = c.at<uint32_t>(c.p.ticket);
    const dim3 grid((unsigned)(T ? c.p.Mpad / 32 : 1));
    rc = dtype == RDB_F32 ? launch_pdl(ce_sum_kernel<float>, grid, 512, 0, c.st, g) : launch_pdl(ce_sum_kernel<__nv_bfloat16>, grid, 512, 0, c.st, g);
    if (rc || T == 0 || !dx_unit) return rc;
    return ce_finish_dx(c, dx_unit, true);
}

extern "C" int rdb_ce_bwd(void *dx, void *dw, const float *dloss, const void *x, int64_t ldx, const void *w, int64_t ldw, const int64_t *target,
                          const float *aux, void *workspace, size_t workspace_bytes, int64_t T, int64_t R, int64_t V, int64_t ignore_index,
                          int use_ignore, int dtype, int reduction, int32_t *status, void *stream) {
    int rc = ce_check(T, R, V, ldx, w, ldw, dtype, reduction);
    if (rc) return rc;
    if (!dx && !dw) return RDB_OK;
    if (T > 0 && (!w || !dloss || !aux || !x || !target)) return RDB_ERR_NULL;
    const size_t es = dtype_size(dtype);
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & (es - 1)) ||
        ((reinterpret_cast<uintptr_t>(dloss) | reinterpret_cast<uintptr_t>(aux)) & 3) || (reinterpret_cast<uintptr_t>(target) & 7))
        return RDB_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (!dw) return RDB_OK;
        cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)V * R * es, st);
        return e == cudaSuccess ? RDB_OK : (int)e;
    }
    CeCall c{};
    c.p = ce_plan(2, T, R, V, dtype, w, ldw, dw, dx ? 1 : 0, dw ? 1 : 0);
    if (!workspace || workspace_bytes < c.p.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return RDB_ERR_WORKSPACE;
    c.ws = reinterpret_cast<uint8_t *>(workspace);
    c.x = x; c.ldx = ldx; c.T = T; c.R = R; c.V = V;
    c.voc = Vocab{w, ldw, 0, 0};
    c.target = target;
    c.dtype = dtype;
    c.status = status;
    c.st = st;
    if ((rc = ce_find_rows(c, ignore_index, use_ignore, nullptr, nullptr, nullptr, nullptr))) return rc;
    CeRowArgs ra = ce_row_args(c);
    ra.dloss = dloss;
    ra.lse = aux;
    ra.loss = aux + T;
    ra.reduction = reduction;
    if ((rc = ce_gather(c, ra))) return rc;
    for (int64_t i = 0; i < c.p.npieces; ++i) {
        const int64_t v0 = i * c.p.piece, n = V - v0 < c.p.piece ? V - v0 : c.p.piece;
        const void *b;
        int64_t ldb;
        if ((rc = ce_stage(c, v0, n, &b, &ldb))) return rc;
        if ((rc = ce_logits<EPI_PROB>(c, b, ldb, v0, n, i))) return rc;
        if (dx && (rc = ce_accumulate(c, b, ldb, n, i > 0))) return rc;
        if (dw && (rc = ce_dw(c, dw, v0, n))) return rc;
    }
    if (dx) return ce_finish_dx(c, dx, false);
    return RDB_OK;
}

extern "C" int rdb_ce_scale(void *dz, const float *unit, const float *dloss, const float *aux, int64_t T, int64_t R, int dtype, int reduction,
                            void *stream) {
    int rc = ce_check(T, R, 1, R, nullptr, 0, dtype, reduction);
    if (rc) return rc;
    if (T == 0) return RDB_OK;
    if (!dz || !unit || !dloss || !aux) return RDB_ERR_NULL;
    if ((reinterpret_cast<uintptr_t>(dz) & (dtype_size(dtype) - 1)) ||
        ((reinterpret_cast<uintptr_t>(unit) | reinterpret_cast<uintptr_t>(dloss) | reinterpret_cast<uintptr_t>(aux)) & 3))
        return RDB_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t want = cdiv64(T * R, 256 * 8);
    const dim3 grid((unsigned)(want < 148 * 8 ? want : 148 * 8));
    if (dtype == RDB_F32)
        return launch_pdl(ce_scale_kernel<float>, grid, 256, 0, st, (float *)dz, unit, dloss, aux + 2 * T, T, R, reduction);
    return launch_pdl(ce_scale_kernel<__nv_bfloat16>, grid, 256, 0, st, (__nv_bfloat16 *)dz, unit, dloss, aux + 2 * T, T, R, reduction);
}
