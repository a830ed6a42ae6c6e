// Linear and gated projections, tiles of 64 WP (P) by 16 NJ WQ (Q): WP x WQ waves of 64 by
// 16 NJ, KG groups of which take the K steps in turn; both operands by buffer DMA into NST
// stages of LDS, NST steps (of every group) ahead.
//
//   Small  64 x 64, 4 waves, 4 stages (64 KB)
//   Deep   128 x 128, one tile per CU (128 KB): 8 waves and 4 stages where k is contiguous;
//          2 groups of 4 waves and 2 stages where an operand lies by columns, as a transposing
//          read brings half as much and waves of 64 x 64 read less (a contraction of 9482 into
//          1024 x 4096: 100 us with 8 waves, 84 with the groups; k contiguous, 1024 x 4096 x
//          4096: 37 and 40)
//   Pair   128 x 128, 4 waves, 2 stages (64 KB): two workgroups per CU, one's epilogue and
//          waits under the other's MFMAs
//   Tall   128 (P) x 256 (Q), 8 waves, 3 stages (144 KB), k contiguous: three quarters of
//          Pair's operand bytes
//
// Where each is taken, and what it measured, stands at cost() in linear.hip.  At their best, bf16:
// Tall 1.15 PFLOP/s (2048 x 4096 x 4096), Pair 0.90 (dx of 9482 x 2304 x 768; MFMA busy 27 % of the
// time), Deep 0.60 (1024 x 4096 x 1024).  What bounds them is neither LDS (a quarter of its cycles
// at most, no bank conflicts) nor the way from L2 (32 KB to a CU take 0.25 to 0.32 us with all CUs
// reading, against 0.54 us for a step of Deep's), which leaves the step's barrier: a wave's MFMAs
// are a quarter of the step, and all waves wait for the last one's reads and loads.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "linear.hpp"

using namespace lin;

namespace {

template <class T, int LAYOUT, int EPI, int WP, int WQ, int NJ, int KG, int NST>
__global__ __launch_bounds__(64 * WP * WQ * KG) __attribute__((amdgpu_waves_per_eu(2))) void linear_tile_kernel(LinearArgs a) {
    constexpr int TP = 64 * WP, TQ = 16 * NJ * WQ;                       // operand rows of a tile
    constexpr int SUB = (TP + TQ) * STEP_BYTES, STAGE = KG * SUB, Q_AT = TP * STEP_BYTES;
    constexpr int PI = 8 / WQ, QI = 2 * NJ / WP;                         // 1 KB DMA instructions per wave and stage
    constexpr bool P_COLS = LAYOUT != ROWS_ROWS, Q_COLS = LAYOUT == COLS_COLS;
    constexpr int ES = T::bytes;
    constexpr int PW = EPI == EPI_GATED ? TP / 2 : TP;                   // output columns of a tile
    __shared__ __align__(1024) uint8_t smem[NST * STAGE];
    const int lane = threadIdx.x & 63, wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave_id / (WP * WQ), wave = wave_id % (WP * WQ);
    const int wp = wave % WP, wq = wave / WP;
    const int n_p = (a.p_cols + PW - 1) / PW, n_q = (a.q_rows + TQ - 1) / TQ;
    int tp, tq;
    tile_coords(blockIdx.x, n_p, n_q, tp, tq);
    const int p0 = tp * PW, q0 = tq * TQ;

    // Sources.  k contiguous: one resource per tile, whose end makes rows past the operand's
    // last read zeros, a byte offset per lane, and the K step as scalar offset.  k as row
    // index: the resource moves down by STEP_ROWS rows each step (see issue).
    const uint8_t* const pb = (const uint8_t*)a.p + (P_COLS ? (long)p0 : (long)p0 * a.ldp) * ES;
    const uint8_t* const qb = (const uint8_t*)a.q + (Q_COLS ? (long)q0 : (long)q0 * a.ldq) * ES;
    const int p_rows = EPI == EPI_GATED ? 2 * a.p_cols - p0 : a.p_cols - p0;
    i32x4 rp, rq;
    if constexpr (!P_COLS) rp = bounded_rsrc(pb, ((long)(p_rows - 1) * a.ldp + a.k) * ES);
    if constexpr (!Q_COLS) rq = bounded_rsrc(qb, ((long)(a.q_rows - q0 - 1) * a.ldq + a.k) * ES);
    uint32_t poff[PI], qoff[QI], pk[PI], qk[QI];
#pragma unroll
    for (int j = 0; j < PI; ++j) {
        const int i = wave * PI + j, r = i * 8 + (lane >> 3), k = (i * 64 + lane) / (TP / 8);
        const int q = (lane % (TP / 8)) ^ col_swz<TP>(k);
        pk[j] = ((lane & 7) ^ row_swz(r)) * 16;
        poff[j] = P_COLS ? (uint32_t)((k * a.ldp + q * 8) * ES) : (uint32_t)(p_row<EPI>(r, a.p_cols) * a.ldp * ES + pk[j]);
    }
#pragma unroll
    for (int j = 0; j < QI; ++j) {
        const int i = wave * QI + j, r = i * 8 + (lane >> 3), k = (i * 64 + lane) / (TQ / 8);
        const int q = (lane % (TQ / 8)) ^ col_swz<TQ>(k);
        qk[j] = ((lane & 7) ^ row_swz(r)) * 16;
        qoff[j] = Q_COLS ? (uint32_t)((k * a.ldq + q * 8) * ES) : (uint32_t)(r * a.ldq * ES + qk[j]);
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem) + kg * SUB;
    const uint32_t kbytes = (uint32_t)a.k * ES;
    const int steps = P_COLS ? (a.k + STEP_ROWS - 1) / STEP_ROWS : (int)((kbytes + STEP_BYTES - 1) / STEP_BYTES);
    const int split = blockIdx.y, kt0 = min(split * a.split_steps, steps), kt1 = min(kt0 + a.split_steps, steps);
    // Loads of step kt into stage st, one instruction at a time.  Steps past the last are zeros
    // (their loads keep the count).
    struct Load {
        bool live;
        uint32_t kb;
        i32x4 rp, rq;
    };
    auto load_of = [&](int kt) {
        Load l;
        l.live = kt < kt1;
        l.kb = l.live ? (uint32_t)kt * STEP_BYTES : 0;  // never past a resource's end
        const long row = (long)kt * STEP_ROWS;
        if constexpr (P_COLS) l.rp = bounded_rsrc(pb + row * a.ldp * ES, l.live ? ((a.k - row - 1) * a.ldp + a.p_cols - p0) * ES : 0);
        else l.rp = rp;
        if constexpr (Q_COLS) l.rq = bounded_rsrc(qb + row * a.ldq * ES, l.live ? ((a.k - row - 1) * a.ldq + a.q_rows - q0) * ES : 0);
        else l.rq = rq;
        return l;
    };
    auto issue = [&](const Load& l, int st, int i) {  // i < PI + QI
        if (i < PI) {
            const uint32_t to = lds0 + st * STAGE + (wave * PI + i) * 1024;
            if constexpr (P_COLS) dma16(to, poff[i], l.rp, 0);
            else dma16(to, l.live && l.kb + pk[i] < kbytes ? poff[i] : OOB, l.rp, l.kb);
        } else {
            const int j = i - PI;
            const uint32_t to = lds0 + st * STAGE + Q_AT + (wave * QI + j) * 1024;
            if constexpr (Q_COLS) dma16(to, qoff[j], l.rq, 0);
            else dma16(to, l.live && l.kb + qk[j] < kbytes ? qoff[j] : OOB, l.rq, l.kb);
        }
    };

    // Where registers are free for it, the epilogue's operands come in before the loop.
    Epilogue<T, LAYOUT, EPI, NJ, NJ, KG == 1 && NJ <= 2> epilogue(a, q0 + wq * 16 * NJ, p0 + wp * (EPI == EPI_GATED ? 32 : 64),
                                                                 lane);
    epilogue.start();
    f32x4 acc[4][NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    const FragReader<T, P_COLS, 4, TP> p_reader(smem + kg * SUB, wp * 64, lane);
    const FragReader<T, Q_COLS, NJ, TQ> q_reader(smem + kg * SUB + Q_AT, wq * 16 * NJ, lane);

    // Step i (of this wave's group): its fragments are in registers and step i + 1 has landed for
    // this wave; past the barrier that holds for everyone, so the fragments of step i + 1 are
    // read, and the loads of step i + NST take the stage that step i leaves, under the
    // multiplications of step i.  In pairs, as the two sets of registers change places: an odd
    // number of steps ends with one of zeros.
    typename decltype(p_reader)::Raw pf[2][4];
    typename decltype(q_reader)::Raw qf[2][NJ];
    auto read = [&](int set, int st, int i) {  // i < 4 + NJ
        if (i < 4) pf[set][i] = p_reader.read(st * STAGE, i);
        else qf[set][i - 4] = q_reader.read(st * STAGE, i - 4);
    };
    int st = 0;  // stage of step i
    auto step = [&](int i, auto parity) {
        constexpr int set = decltype(parity)::value, READS = 4 + NJ, LOADS = PI + QI, TILES = 4 * NJ;
        const int next = st + 1 == NST ? 0 : st + 1;
        const Load l = load_of(kt0 + (i + NST) * KG + kg);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NST - 2) * LOADS) : "memory");
        // Reads and loads go out between the multiplications, which leave the wave free to issue
        // them; with two workgroups on a CU they go first, the other's multiplications covering
        // them (128 x 128 tiles, K = 4096: 33 -> 27 us for 32 tiles one to a CU, but 60 -> 63 us
        // for 512 of them two to a CU).
        constexpr int SPAN = NST > 2 || KG > 1 ? TILES : 1;
#pragma unroll
        for (int m = 0; m < TILES; ++m) {
#pragma unroll
            for (int r = 0; r < READS; ++r)
                if (r * SPAN / READS == m) read(set ^ 1, next, r);
#pragma unroll
            for (int r = 0; r < LOADS; ++r)
                if (r * SPAN / LOADS == m) issue(l, st, r);
            acc[m % 4][m / 4] = T::mfma(pf[set][m % 4].frag(), qf[set][m / 4].frag(), acc[m % 4][m / 4]);
            if (SPAN > 1 || m == 0) __builtin_amdgcn_sched_barrier(0);
        }
        st = next;
    };
#pragma unroll
    for (int s = 0; s < NST; ++s) {
        const Load l = load_of(kt0 + s * KG + kg);
#pragma unroll
        for (int i = 0; i < PI + QI; ++i) issue(l, s, i);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NST - 1) * (PI + QI)) : "memory");
#pragma unroll
    for (int i = 0; i < 4 + NJ; ++i) read(0, 0, i);
    const int n = (kt1 - kt0 + KG - 1) / KG;
    for (int i = 0; i < n; i += 2) {
        step(i, std::integral_constant<int, 0>{});
        step(i + 1, std::integral_constant<int, 1>{});
    }
    // No load may still be on its way into LDS when it is used again, or the workgroup ends.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

    // The groups' sums are added in group order.
    if constexpr (KG > 1) {
        f32x4* const sums = (f32x4*)smem + wave * (4 * NJ * 64) + lane;
        constexpr int GROUP = WP * WQ * 4 * NJ * 64;
        __syncthreads();
        if (kg) {
#pragma unroll
            for (int i = 0; i < 4 * NJ; ++i) sums[(kg - 1) * GROUP + i * 64] = acc[i / NJ][i % NJ];
        }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int g = 0; g < KG - 1; ++g)
#pragma unroll
            for (int i = 0; i < 4 * NJ; ++i) acc[i / NJ][i % NJ] += sums[g * GROUP + i * 64];
    }

    epilogue.finish(acc, split);
}

template <class T, int LAYOUT, int EPI, int WP, int WQ, int NJ, int KG, int NST>
void launch_tiles(const LinearArgs& a, hipStream_t s) {
    const long pw = EPI == EPI_GATED ? 32 * WP : 64 * WP, qw = 16 * NJ * WQ;
    const long tiles = ((a.p_cols + pw - 1) / pw) * ((a.q_rows + qw - 1) / qw);
    if (tiles * 64L * WP * WQ * KG >= 1L << 32) throw jh_error(JH_ERR_INVALID, "linear: too many tiles");
    JH_LAUNCH((linear_tile_kernel<T, LAYOUT, EPI, WP, WQ, NJ, KG, NST>), dim3((unsigned)tiles, (unsigned)a.splits),
              dim3(64 * WP * WQ * KG), 0, s, a);
    HIP_CHECK(hipGetLastError());
}

template <class T, int LAYOUT, int EPI>
void launch(const LinearArgs& a, LinearTile tile, hipStream_t s) {
    if (tile == LinearTile::Small) launch_tiles<T, LAYOUT, EPI, 1, 4, 1, 1, 4>(a, s);
    else if (tile == LinearTile::Pair) launch_tiles<T, LAYOUT, EPI, 2, 2, 4, 1, 2>(a, s);
    else if constexpr (LAYOUT != ROWS_ROWS) {
        launch_tiles<T, LAYOUT, EPI, 2, 2, 4, 2, 2>(a, s);
    } else if (std::is_same_v<T, E4m3Wide> || tile == LinearTile::Deep) launch_tiles<T, LAYOUT, EPI, 2, 4, 2, 1, 4>(a, s);
    else if constexpr (!std::is_same_v<T, E4m3Wide>) launch_tiles<T, LAYOUT, EPI, 2, 4, 4, 1, 3>(a, s);
}

}  // namespace

void launch_linear_tile(const LinearArgs& a, LinearTile tile, hipStream_t s) {
    if (a.gated) {
        if (a.type == JH_BF16) launch<Bf16, ROWS_ROWS, EPI_GATED>(a, tile, s);
        else if (a.type == JH_F16) launch<F16, ROWS_ROWS, EPI_GATED>(a, tile, s);
        else launch<E4m3, ROWS_ROWS, EPI_GATED>(a, tile, s);
    } else if (a.type == JH_E4M3) {
        if (a.out_f32) launch<E4m3Wide, ROWS_ROWS, EPI_LINEAR>(a, tile, s);
        else launch<E4m3, ROWS_ROWS, EPI_LINEAR>(a, tile, s);
    } else if (a.type == JH_BF16) {
        if (a.layout == ROWS_ROWS) launch<Bf16, ROWS_ROWS, EPI_LINEAR>(a, tile, s);
        else if (a.layout == COLS_ROWS) launch<Bf16, COLS_ROWS, EPI_LINEAR>(a, tile, s);
        else launch<Bf16, COLS_COLS, EPI_LINEAR>(a, tile, s);
    } else {
        if (a.layout == ROWS_ROWS) launch<F16, ROWS_ROWS, EPI_LINEAR>(a, tile, s);
        else if (a.layout == COLS_ROWS) launch<F16, COLS_ROWS, EPI_LINEAR>(a, tile, s);
        else launch<F16, COLS_COLS, EPI_LINEAR>(a, tile, s);
    }
}
