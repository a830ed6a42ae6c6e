// Linear and gated projections, 256 x 256 tiles: eight waves of 128 (P) x 64 (Q), one
// workgroup per CU.  Against 128 x 128 tiles this halves the operand bytes that L2 and the
// LDS DMA move per MFMA.
//
// Measured (MFMA busy and clock from counters): 16384 x 8192 x 2048 bf16 gated with silu and both
// projections kept, 1.10 PFLOP in 891 us (1.23 PFLOP/s, busy 59 % at 1.91 GHz: power holds the
// clock there, 2.4 GHz at rest); 8192 x 4096 x 4096 bf16 200 us (1.37); 4096^3 e4m3 57 us (2.40);
// 8192 x 4096 x 4096 e4m3 105 us (2.6), with bias, silu and residual 122 to 128 (2.2): all tiles of a
// round end together, 67 MB of residuals and outputs in a burst, twice.  LDS is read a fifth of
// the time, without bank conflicts; a step's 64 KB of operands take half as long to come in as its
// MFMAs (2048 cycles), all CUs reading.
//
// A K step runs in four phases, each a quadrant of the wave's block: 64 P rows by 32 Q rows,
// 16 MFMAs of 16 bits.  A phase first reads the fragments that it or the next lacks and
// issues one part of the operands two K steps ahead, then meets a barrier, multiplies, and
// meets another.  f is the Q half that the step multiplies first, s the other; they change
// places every step, so that the half whose registers are free in the last phase is the one
// that the next step begins with:
//
//   phase   reads          multiplies   issues (part of step t + 2)
//   0       Pa             Pa x Qf      Qf
//   1       Qs             Pa x Qs      Pa
//   2       Pb             Pb x Qs      Qs
//   3       Qs of t + 1    Pb x Qf      Pb
//
// The two waves of a SIMD (w and w + 4) run one half phase apart, waves 4-7 having met one
// barrier more: while one multiplies, the other reads and issues.
//
// LDS holds two K steps of four 16 KB parts, two of either operand.  Q's hold its first and last
// 128 rows (columns, where k is the row index), 32 of each for a wave.  P's: by columns the first
// and last 128, 64 of each for a wave (one run of 256 bytes per k; when this was chosen the weight
// gradient of 29367 x 3464 x 1504, now 283 us in parts, took 403 so and 426 in runs of 64 and 128); by rows the first and last 64 of a
// wave's 128 (16384 x 4096 x 512: 91 us, 94 with the halves 128 apart); gated the gate's 128 rows
// and the up projection's.  So a lane ends with 16 consecutive output columns and four lanes with
// 64 of a row, whatever the layout: the epilogue writes whole 128-byte lines.  A part read in
// one phase is refilled in the next: every wave has waited for its own reads (lgkmcnt) before
// the barrier that the refilling waves have passed.  A part is read seven phases after its
// issue, and one phase after every wave has waited for its own share of it: a wave issues two
// loads per phase, six phases' worth after that part, hence vmcnt(12).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "linear.hpp"

using namespace lin;

namespace {

constexpr int TILE = 256, PART = 16384;
enum { PA, PB, QA, QB };
// Both stages of an operand lie within the 64 KB that an LDS read's offset spans.
__device__ constexpr int part_at(int st, int part) { return ((part >> 1) * 4 + st * 2 + (part & 1)) * PART; }

// Epilogue of a wave's 64 gate and up columns (16 of each per lane, from c) and 64 rows from t0.
template <class T>
__device__ inline void finish_gated(const LinearArgs& a, const f32x4 (&acc)[2][4][4], int t0, int c, int lane) {
    ColumnTerms<T> gate[2], up[2];
    if constexpr (T::bytes == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            gate[h].load(a, c + 8 * h, a.p_scale);
            up[h].load(a, c + 8 * h, a.p_scale ? a.p_scale + a.p_cols : nullptr);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long first = t0 + (j & 1) * 16 + (j >> 1) * 128;
        float g[2][8], u[2][8];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            g[e >> 3][e & 7] = acc[0][e >> 2][j][e & 3];
            u[e >> 3][e & 7] = acc[1][e >> 2][j][e & 3];
        }
        if constexpr (T::bytes == 1) {
            const float qs = a.q_scale ? a.q_scale[min(first + (lane & 15), (long)a.q_rows - 1)] : 1.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                gate[h].apply(a, g[h], qs);
                up[h].apply(a, u[h], qs);
            }
        } else if (a.pre) {
            store_half<T>(a.pre, a.ldpre, first, c, lane, a.q_rows, a.p_cols, g);
            store_half<T>((uint16_t*)a.pre + a.p_cols, a.ldpre, first, c, lane, a.q_rows, a.p_cols, u);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            activate(g[h], a.act);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[h][e] *= u[h][e];
        }
        store_half<T>(a.out, a.ldo, first, c, lane, a.q_rows, a.p_cols, g);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <class T, int LAYOUT, int EPI>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void linear_wide_kernel(LinearArgs a) {
    constexpr bool P_COLS = LAYOUT != ROWS_ROWS, Q_COLS = LAYOUT == COLS_COLS;
    constexpr int ES = T::bytes;
    constexpr int PW = EPI == EPI_GATED ? TILE / 2 : TILE;
    __shared__ __align__(1024) uint8_t smem[8 * PART];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wp = wave >> 2, wq = wave & 3;
    const int n_p = (a.p_cols + PW - 1) / PW, n_q = (a.q_rows + TILE - 1) / TILE;
    int tp, tq;
    tile_coords(blockIdx.x, n_p, n_q, tp, tq);
    const int p0 = tp * PW, q0 = tq * TILE;

    // Sources, as in linear_tile_kernel, with one offset per lane and instruction for both
    // halves of an operand: the second half lies p_half (q_half) bytes further.
    const uint8_t* const pb = (const uint8_t*)a.p + (P_COLS ? (long)p0 : (long)p0 * a.ldp) * ES;
    const uint8_t* const qb = (const uint8_t*)a.q + (Q_COLS ? (long)q0 : (long)q0 * a.ldq) * ES;
    const long p_half = P_COLS ? 128 * ES : (EPI == EPI_GATED ? (long)a.p_cols : 64L) * a.ldp * ES;
    const long q_half = (Q_COLS ? 128L : 128 * a.ldq) * ES;
    const int p_rows = EPI == EPI_GATED ? 2 * a.p_cols - p0 : a.p_cols - p0;
    const long p_bytes = ((long)(p_rows - 1) * a.ldp + a.k) * ES, q_bytes = ((long)(a.q_rows - q0 - 1) * a.ldq + a.k) * ES;
    i32x4 rp[2], rq[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (!P_COLS) rp[h] = bounded_rsrc(pb + h * p_half, p_bytes - h * p_half);
        if constexpr (!Q_COLS) rq[h] = bounded_rsrc(qb + h * q_half, q_bytes - h * q_half);
    }
    uint32_t poff[2], qoff[2];
    const uint32_t kbytes = (uint32_t)a.k * ES;
    const int steps = P_COLS ? (a.k + STEP_ROWS - 1) / STEP_ROWS : (int)((kbytes + STEP_BYTES - 1) / STEP_BYTES);
    uint64_t tail[2];  // lanes whose chunk of a k-contiguous row the last step still has
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = (wave * 2 + j) * 8 + (lane >> 3);               // row of a k-contiguous part
        const int k = (wave * 2 + j) * 4 + (lane >> 4), q = (lane & 15) ^ col_swz<128>(k);  // row and chunk of a part by columns
        const uint32_t rk = ((lane & 7) ^ row_swz(r)) * 16;
        tail[j] = __builtin_amdgcn_ballot_w64((steps - 1) * STEP_BYTES + rk < kbytes);
        poff[j] = P_COLS ? (uint32_t)((k * a.ldp + q * 8) * ES)
                         : (uint32_t)((p_row<EPI_LINEAR>(r, 0) + (EPI == EPI_GATED ? 0 : r & 64)) * a.ldp * ES + rk);
        qoff[j] = Q_COLS ? (uint32_t)((k * a.ldq + q * 8) * ES) : (uint32_t)(r * a.ldq * ES + rk);
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)&smem[wave * 2048]);
    const int split = blockIdx.y, kt0 = min(split * a.split_steps, steps), kt1 = min(kt0 + a.split_steps, steps);
    // Parts past the last step are zeros (their loads keep the count).
    auto issue = [&](int part, int kt, int st) {
        const bool p = part < QA, live = kt < kt1;
        const int h = part & 1;
        const uint32_t kb = live ? (uint32_t)kt * STEP_BYTES : 0;  // never past the resource's end
        i32x4 r = p ? rp[h] : rq[h];
        if (p ? P_COLS : Q_COLS) {
            const long ld = p ? a.ldp : a.ldq, cols = p ? a.p_cols - p0 : a.q_rows - q0;
            const long row = (long)kt * STEP_ROWS, half = h * (p ? p_half : q_half);
            r = bounded_rsrc((p ? pb : qb) + row * ld * ES + half, live ? ((a.k - row - 1) * ld + cols) * ES - half : 0);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t l = lds0 + part_at(st, part) + j * 1024, off = p ? poff[j] : qoff[j];
            if (p ? P_COLS : Q_COLS) dma16(l, off, r, 0);
            else dma16(l, __builtin_amdgcn_inverse_ballot_w64(!live ? 0 : kt < steps - 1 ? ~0ull : tail[j]) ? off : OOB, r, kb);
        }
    };

    f32x4 acc[2][4][4];  // P half, P tile, Q tile
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][i][j] = f32x4{0, 0, 0, 0};
    typename T::Frag pf[4], qf[4];

    // Step t is kt0 + t; its stage is t % 2, and the Q half it multiplies first is a for even t,
    // b for odd.
    issue(QA, kt0, 0);
    issue(PA, kt0, 0);
    issue(QB, kt0, 0);
    issue(PB, kt0, 0);
    issue(QB, kt0 + 1, 1);
    issue(PA, kt0 + 1, 1);
    issue(QA, kt0 + 1, 1);
    issue(PB, kt0 + 1, 1);
    asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier" ::: "memory");
    const FragReader<T, P_COLS, 4> p_reader(smem + part_at(0, PA), wp * 64, lane);
    const FragReader<T, Q_COLS, 2> q_reader(smem + part_at(0, QA), wq * 32, lane);
    auto read_p = [&](int st, int h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[i] = p_reader.read(part_at(st, PA + h) - part_at(0, PA), i).frag();
    };
    auto read_q = [&](int st, int h) {
#pragma unroll
        for (int j = 0; j < 2; ++j) qf[h * 2 + j] = q_reader.read(part_at(st, QA + h) - part_at(0, QA), j).frag();
    };
    // One quadrant: P half ph by Q half qh.
    auto multiply = [&](int ph, int qh) {
        asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[ph][i][qh * 2 + j] = T::mfma(pf[i], qf[qh * 2 + j], acc[ph][i][qh * 2 + j]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
    };
    auto step = [&](int kt, auto parity) {
        constexpr int st = decltype(parity)::value, first = st, second = st ^ 1;
        read_p(st, 0);
        issue(QA + first, kt + 2, st);
        multiply(0, first);
        read_q(st, second);
        issue(PA, kt + 2, st);
        multiply(0, second);
        read_p(st, 1);
        issue(QA + second, kt + 2, st);
        multiply(1, second);
        read_q(st ^ 1, second);  // the next step's first half
        issue(PB, kt + 2, st);
        multiply(1, first);
    };
    // Every wave has read its first half before any refills it.
    read_q(0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (wp) asm volatile("s_barrier" ::: "memory");
    // In pairs: an odd number of steps ends with one of zeros.
    for (int kt = kt0; kt < kt1; kt += 2) {
        step(kt, std::integral_constant<int, 0>{});
        step(kt + 1, std::integral_constant<int, 1>{});
    }
    if (!wp) asm volatile("s_barrier" ::: "memory");
    // No load may still be on its way into LDS when the workgroup ends.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    // The second half of the wave's Q rows lies 128 rows on.
    const int t0 = q0 + wq * 32;
    const int l = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));  // `lane`, not kept over the loop
    if constexpr (EPI == EPI_GATED) {
        finish_gated<T>(a, acc, t0, p0 + wp * 64 + (l >> 4) * 16, l);
    } else {
        const int first = p0 + wp * (P_COLS ? 64 : 128), second = first + (P_COLS ? 128 : 64);
        Epilogue<T, LAYOUT, EPI, 4, 2, false>(a, t0, first, l).finish(acc[0], split);
        __builtin_amdgcn_sched_barrier(0);
        Epilogue<T, LAYOUT, EPI, 4, 2, false>(a, t0, second, l).finish(acc[1], split);
    }
}

template <class T, int LAYOUT, int EPI>
void launch(const LinearArgs& a, hipStream_t s) {
    const long pw = EPI == EPI_GATED ? TILE / 2 : TILE;
    const long tiles = ((a.p_cols + pw - 1) / pw) * ((a.q_rows + TILE - 1L) / TILE);
    if (tiles * 512 >= 1L << 32) throw jh_error(JH_ERR_INVALID, "linear: too many tiles");
    JH_LAUNCH((linear_wide_kernel<T, LAYOUT, EPI>), dim3((unsigned)tiles, (unsigned)a.splits), dim3(512), 0, s, a);
    HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_linear_wide(const LinearArgs& a, hipStream_t s) {
    if (a.gated) {
        if (a.type == JH_BF16) launch<Bf16, ROWS_ROWS, EPI_GATED>(a, s);
        else if (a.type == JH_F16) launch<F16, ROWS_ROWS, EPI_GATED>(a, s);
        else launch<E4m3, ROWS_ROWS, EPI_GATED>(a, s);
    } else if (a.type == JH_E4M3) {
        launch<E4m3, ROWS_ROWS, EPI_LINEAR>(a, s);
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
