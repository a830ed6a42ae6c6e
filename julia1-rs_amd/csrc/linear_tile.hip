// Linear and gated projections, 128 x 128 tiles: four waves of 64 x 64, both operands by
// buffer DMA into two 32 KB stages of LDS, two workgroups per CU (one's epilogue and waits
// run under the other's MFMAs).
#include <hip/hip_runtime.h>

#include "linear.hpp"

using namespace lin;

namespace {

template <class T, int LAYOUT, int EPI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void linear_tile_kernel(LinearArgs a) {
    constexpr int TILE = 128, PART = TILE * STEP_BYTES, IPW = 4;  // 1 KB DMA instructions per wave, operand and stage
    constexpr bool P_COLS = LAYOUT != ROWS_ROWS, Q_COLS = LAYOUT == COLS_COLS;
    constexpr int ES = T::bytes;
    __shared__ __align__(1024) uint8_t smem[4 * PART];
    uint8_t* const sP = smem;
    uint8_t* const sQ = smem + 2 * PART;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int PW = EPI == EPI_GATED ? TILE / 2 : TILE;  // output columns of a tile
    const int n_p = (a.p_cols + PW - 1) / PW, n_q = (a.q_rows + TILE - 1) / TILE;
    int tp, tq;
    tile_coords(blockIdx.x, n_p, n_q, tp, tq);
    const int p0 = tp * PW, q0 = tq * TILE;

    // Sources.  k contiguous: one resource per tile, whose end makes rows past the operand's
    // last read zeros, a byte offset per lane, and the K step as scalar offset.  k as row
    // index: the resource moves down by STEP_ROWS rows each step (see issue).
    const uint8_t* const pb = (const uint8_t*)a.p + (P_COLS ? (long)p0 : (long)p0 * a.ldp) * ES;
    const uint8_t* const qb = (const uint8_t*)a.q + (Q_COLS ? (long)q0 : (long)q0 * a.ldq) * ES;
    const int p_rows = EPI == EPI_GATED ? 2 * a.p_cols - p0 : a.p_cols - p0;
    i32x4 rp, rq;
    if constexpr (!P_COLS) rp = bounded_rsrc(pb, ((long)(p_rows - 1) * a.ldp + a.k) * ES);
    if constexpr (!Q_COLS) rq = bounded_rsrc(qb, ((long)(a.q_rows - q0 - 1) * a.ldq + a.k) * ES);
    uint32_t poff[IPW], qoff[IPW], pk[IPW], qk[IPW];
#pragma unroll
    for (int j = 0; j < IPW; ++j) {
        const int rr = (wave * IPW + j) * 8 + (lane >> 3), rk = ((lane & 7) ^ row_swz(rr)) * 16;
        const int cr = (wave * IPW + j) * 4 + (lane >> 4), cc = ((lane & 15) ^ col_swz(cr)) * 16;
        pk[j] = qk[j] = (uint32_t)rk;
        poff[j] = P_COLS ? (uint32_t)(cr * a.ldp * ES + cc) : (uint32_t)(p_row<EPI>(rr, a.p_cols) * a.ldp * ES + rk);
        qoff[j] = Q_COLS ? (uint32_t)(cr * a.ldq * ES + cc) : (uint32_t)(rr * a.ldq * ES + rk);
    }
    const uint32_t pl0 = (uint32_t)(uintptr_t)&sP[wave * IPW * 1024], ql0 = (uint32_t)(uintptr_t)&sQ[wave * IPW * 1024];
    const uint32_t kbytes = (uint32_t)a.k * ES;
    auto issue = [&](int kt, int st) {
        if constexpr (P_COLS)
            rp = bounded_rsrc(pb + (long)kt * STEP_ROWS * a.ldp * ES,
                              ((long)(a.k - kt * STEP_ROWS - 1) * a.ldp + a.p_cols - p0) * ES);
        if constexpr (Q_COLS)
            rq = bounded_rsrc(qb + (long)kt * STEP_ROWS * a.ldq * ES,
                              ((long)(a.k - kt * STEP_ROWS - 1) * a.ldq + a.q_rows - q0) * ES);
        const uint32_t kb = (uint32_t)kt * STEP_BYTES;
#pragma unroll
        for (int j = 0; j < IPW; ++j) {
            const uint32_t lp = __builtin_amdgcn_readfirstlane(pl0 + st * PART + j * 1024);
            const uint32_t lq = __builtin_amdgcn_readfirstlane(ql0 + st * PART + j * 1024);
            if constexpr (P_COLS) dma16(lp, poff[j], rp, 0);
            else dma16(lp, kb + pk[j] < kbytes ? poff[j] : OOB, rp, kb);
            if constexpr (Q_COLS) dma16(lq, qoff[j], rq, 0);
            else dma16(lq, kb + qk[j] < kbytes ? qoff[j] : OOB, rq, kb);
        }
    };

    const int wp = wave & 1, wq = wave >> 1;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    const int steps = P_COLS ? (a.k + STEP_ROWS - 1) / STEP_ROWS : (int)((kbytes + STEP_BYTES - 1) / STEP_BYTES);
    const int split = blockIdx.y, kt0 = min(split * a.split_steps, steps), kt1 = min(kt0 + a.split_steps, steps);
    if (kt0 < kt1) issue(kt0, 0);
    for (int kt = kt0; kt < kt1; ++kt) {
        const int st = (kt - kt0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (kt + 1 < kt1) issue(kt + 1, st ^ 1);
        const uint8_t* P = sP + st * PART;
        const uint8_t* Q = sQ + st * PART;
        typename T::Frag pf[4], qf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pf[i] = frag<T, P_COLS>(P, wp * 64 + i * 16, lane);
            qf[i] = frag<T, Q_COLS>(Q, wq * 64 + i * 16, lane);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = T::mfma(pf[i], qf[j], acc[i][j]);
    }

    const int col0 = p0 + wp * (EPI == EPI_GATED ? 32 : 64);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f32x4 c[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
        finish_block<T, LAYOUT, EPI>(a, c, q0 + wq * 64 + j * 16, col0, lane, split);
    }
}

template <class T, int LAYOUT, int EPI>
void launch(const LinearArgs& a, hipStream_t s) {
    const long pw = EPI == EPI_GATED ? 64 : 128;
    const long tiles = ((a.p_cols + pw - 1) / pw) * ((a.q_rows + 127L) / 128);
    if (tiles > 0x7fffffffL) throw jh_error(JH_ERR_INVALID, "linear: too many tiles");
    JH_LAUNCH((linear_tile_kernel<T, LAYOUT, EPI>), dim3((unsigned)tiles, (unsigned)a.splits), dim3(256), 0, s, a);
    HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_linear_tile(const LinearArgs& a, hipStream_t s) {
    if (a.gated) {
        if (a.type == JH_BF16) launch<Bf16, ROWS_ROWS, EPI_GATED>(a, s);
        else if (a.type == JH_F16) launch<F16, ROWS_ROWS, EPI_GATED>(a, s);
        else launch<E4m3, ROWS_ROWS, EPI_GATED>(a, s);
    } else if (a.type == JH_E4M3) {
        if (a.out_f32) launch<E4m3Wide, ROWS_ROWS, EPI_LINEAR>(a, s);
        else launch<E4m3, ROWS_ROWS, EPI_LINEAR>(a, s);
    } else if (a.type == JH_BF16) {
        if (a.layout == ROWS_ROWS) launch<Bf16, ROWS_ROWS, EPI_LINEAR>(a, s);
        else if (a.layout == COLS_ROWS) launch<Bf16, COLS_ROWS, EPI_LINEAR>(a, s);
        else launch<Bf16, COLS_COLS, EPI_LINEAR>(a, s);
    } else {
        if (a.layout == ROWS_ROWS) launch<F16, ROWS_ROWS, EPI_LINEAR>(a, s);
        else if (a.layout == COLS_ROWS) launch<F16, COLS_ROWS, EPI_LINEAR>(a, s);
        else launch<F16, COLS_COLS, EPI_LINEAR>(a, s);
    }
}
