// Linear and gated projections of few rows: W streams from memory straight into registers,
// once per 16 * TB rows of X.  A workgroup of eight waves computes 16 * PT operand rows (PT =
// 1 or 2 blocks of 16 columns; the gate and the up block of 16 columns when gated) for 16 * TB
// rows of X; its waves take the K steps in turn and add their sums through LDS in wave order.
#include <hip/hip_runtime.h>

#include "linear.hpp"

using namespace lin;

namespace {

constexpr int NW = 8;

template <class T, int EPI, int PT, int TB>
__global__ __launch_bounds__(64 * NW) void linear_small_kernel(LinearArgs a) {
    constexpr int ES = T::bytes;
    constexpr int PW = EPI == EPI_GATED ? 16 : 16 * PT;  // output columns of a workgroup
    __shared__ __align__(16) f32x4 sums[NW][PT * TB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, m = lane & 15;
    const int p0 = blockIdx.x * PW, q0 = blockIdx.y * 16 * TB;
    const int kbytes = a.k * ES, steps = (kbytes + STEP_BYTES - 1) / STEP_BYTES;

    // Rows past the operand's end read its last row; those products are not stored.
    const uint8_t *pr[PT], *qr[TB];
#pragma unroll
    for (int i = 0; i < PT; ++i) {
        const long r = min(p0 + (EPI == EPI_GATED ? 0 : 16 * i) + m, a.p_cols - 1) + (EPI == EPI_GATED ? (long)i * a.p_cols : 0L);
        pr[i] = (const uint8_t*)a.p + r * a.ldp * ES;
    }
#pragma unroll
    for (int j = 0; j < TB; ++j) qr[j] = (const uint8_t*)a.q + (long)min(q0 + 16 * j + m, a.q_rows - 1) * a.ldq * ES;

    f32x4 acc[PT][TB];
#pragma unroll
    for (int i = 0; i < PT; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    // Chunks past K are zeros in both operands (a NaN in either would spoil the sum).
    constexpr int U = PT * TB <= 2 ? 4 : 2;  // K steps in flight per wave
    for (int s0 = wave; s0 < steps; s0 += NW * U) {
        u32x4 pf[U][PT][2], qf[U][TB][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = (s0 + u * NW) * STEP_BYTES + h * 64 + g * 16;
                const bool in = at < kbytes;
                const int off = in ? at : 0;
#pragma unroll
                for (int i = 0; i < PT; ++i) {
                    pf[u][i][h] = *(const u32x4*)(pr[i] + off);
                    if (!in) pf[u][i][h] = u32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int j = 0; j < TB; ++j) {
                    qf[u][j][h] = *(const u32x4*)(qr[j] + off);
                    if (!in) qf[u][j][h] = u32x4{0, 0, 0, 0};
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < PT; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j)
                    acc[i][j] = T::mfma(T::make(pf[u][i][0], pf[u][i][1]), T::make(qf[u][j][0], qf[u][j][1]), acc[i][j]);
    }

#pragma unroll
    for (int i = 0; i < PT; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) sums[wave][i * TB + j][lane] = acc[i][j];
    __syncthreads();
    // One output (row, 8 columns) per thread: lanes 0-15 of group g hold columns 4g .. 4g+3,
    // so 8 columns are two neighbouring groups.
    constexpr int BLOCKS = EPI == EPI_GATED ? TB : PT * TB;
    for (int o = threadIdx.x; o < BLOCKS * 32; o += 64 * NW) {
        const int blk = o >> 5, half = (o >> 4) & 1, row = o & 15;
        const int j = blk % TB, i = blk / TB;
        const long t = q0 + 16 * j + row;
        const int c0 = p0 + 16 * i + half * 8;
        if (t >= a.q_rows || c0 >= a.p_cols) continue;
        auto total = [&](int tile, float (&v)[8]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int l = (half * 2 + h) * 16 + row;
                f32x4 s = sums[0][tile][l];
#pragma unroll
                for (int w = 1; w < NW; ++w) s += sums[w][tile][l];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * h + e] = s[e];
            }
        };
        const float qs = ES == 1 && a.q_scale ? a.q_scale[t] : 1.0f;
        if constexpr (EPI == EPI_GATED) {
            float ga[8], up[8];
            total(j, ga);
            total(TB + j, up);
            finish_gated8<T>(a, ga, up, t, c0, qs);
        } else {
            float z[8];
            total(i * TB + j, z);
            finish8<T>(a, z, t, c0, qs);
        }
    }
}

template <class T, int EPI, int PT, int TB>
void launch(const LinearArgs& a, hipStream_t s) {
    const unsigned pw = EPI == EPI_GATED ? 16 : 16 * PT;
    JH_LAUNCH((linear_small_kernel<T, EPI, PT, TB>),
              dim3((unsigned)(a.p_cols + pw - 1) / pw, (unsigned)(a.q_rows + 16 * TB - 1) / (16 * TB)), dim3(64 * NW), 0,
              s, a);
    HIP_CHECK(hipGetLastError());
}

template <class T>
void dispatch(const LinearArgs& a, hipStream_t s) {
    if (a.gated) {
        if (a.q_rows <= 16) launch<T, EPI_GATED, 2, 1>(a, s);
        else if (a.q_rows <= 32) launch<T, EPI_GATED, 2, 2>(a, s);
        else launch<T, EPI_GATED, 2, 4>(a, s);
    } else {
        if (a.q_rows <= 16) launch<T, EPI_LINEAR, 1, 1>(a, s);
        else if (a.q_rows <= 32) launch<T, EPI_LINEAR, 2, 2>(a, s);
        else launch<T, EPI_LINEAR, 2, 4>(a, s);
    }
}

}  // namespace

void launch_linear_small(const LinearArgs& a, hipStream_t s) {
    if (a.type == JH_BF16) dispatch<Bf16>(a, s);
    else if (a.type == JH_F16) dispatch<F16>(a, s);
    else if (a.out_f32) dispatch<E4m3Wide>(a, s);
    else dispatch<E4m3>(a, s);
}
