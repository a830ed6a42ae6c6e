// Linear and gated projections of up to 16 rows: W streams from memory straight into
// registers, once.  A workgroup of eight waves computes 16 output columns (their gate and up
// rows when gated); its waves take pieces of K in turn, several loads in flight, and their sums
// are added through LDS in wave order.  MFMA does the products because the rows come for free
// there, not for its rate; x is read by every workgroup, from L2.
//
// Bound by latency while W is small (a launch is 2 us; W's first bytes come 2 us later): 8 x 1152
// x 768 gated, 3.5 MB, 5.0 us; 1 x 768 x 1152, 1.8 MB, 4.1 us; then by memory: 16 x 4096 x 4096,
// 34 MB, 10.1 us (3.3 TB/s).
#include <hip/hip_runtime.h>

#include "linear.hpp"

using namespace lin;

namespace {

constexpr int NW = 8;

// The residual of eight columns of one row, raw (e4m3 operands with FP32 outputs are E4m3Wide).
template <class T>
struct Resid8 {
    static constexpr bool HALF_ONLY = __is_same(T, E4m3);
    u32x4 v[HALF_ONLY ? 1 : 2];
    __device__ void load(const LinearArgs& a, long t, int c0) {
        const long at = min(t, (long)a.q_rows - 1) * a.ldr + min(c0, a.p_cols - 8);
        if (!HALF_ONLY && a.out_f32) {
            v[0] = *(const u32x4*)((const float*)a.resid + at);
            v[HALF_ONLY ? 0 : 1] = *(const u32x4*)((const float*)a.resid + at + 4);
        } else {
            v[0] = *(const u32x4*)((const uint16_t*)a.resid + at);
        }
    }
};

// Eight columns of one output row from their sums z: c0 .. c0+7.
template <class T>
__device__ inline void finish8(const LinearArgs& a, float (&z)[8], long t, int c0, float qs, const ColumnTerms<T>& col,
                               const Resid8<T>& resid) {
    col.apply(a, z, qs);
    if constexpr (T::bytes == 2)
        if (a.pre) store16<T>((uint16_t*)a.pre + t * a.ldpre + c0, z);
    activate(z, a.act);
    if (!Resid8<T>::HALF_ONLY && a.out_f32) {
        if (a.resid) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t r = resid.v[Resid8<T>::HALF_ONLY ? 0 : e >> 2][e & 3];
                z[e] += __builtin_bit_cast(float, r);
            }
        }
        float* o = (float*)a.out + t * a.ldo + c0;
        *(f32x4*)o = f32x4{z[0], z[1], z[2], z[3]};
        *(f32x4*)(o + 4) = f32x4{z[4], z[5], z[6], z[7]};
    } else {
        if (a.resid) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t r = resid.v[0][e];
                z[2 * e] += T::lo(r);
                z[2 * e + 1] += T::hi(r);
            }
        }
        store16<T>((uint16_t*)a.out + t * a.ldo + c0, z);
    }
}

template <class T, int EPI>
__global__ __launch_bounds__(64 * NW) void linear_small_kernel(LinearArgs a) {
    constexpr int ES = T::bytes, PT = EPI == EPI_GATED ? 2 : 1;  // blocks of 16 P rows
    __shared__ __align__(16) f32x4 sums[NW][PT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, m = lane & 15;
    const int p0 = blockIdx.x * 16;
    const int kbytes = a.k * ES, pieces = (kbytes + 63) / 64;

    // Rows past the operand's end read its last row; those products are not stored.
    const uint8_t* pr[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i)
        pr[i] = (const uint8_t*)a.p + (min(p0 + m, a.p_cols - 1) + (long)i * a.p_cols) * a.ldp * ES;
    const uint8_t* const qr = (const uint8_t*)a.q + (long)min(m, a.q_rows - 1) * a.ldq * ES;

    f32x4 acc[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i) acc[i] = f32x4{0, 0, 0, 0};

    // 64 bytes of every row at a time, which the waves take in turn; chunks past K are zeros in
    // both operands (a NaN in either would spoil the sum).
    constexpr int U = 8;  // loads of each row in flight per wave
    const u32x4 zero = {0, 0, 0, 0};
    for (int s0 = wave; s0 < pieces; s0 += NW * U) {
        u32x4 pf[U][PT], qf[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (s0 + u * NW) * 64 + g * 16;
            qf[u] = zero;
#pragma unroll
            for (int i = 0; i < PT; ++i) pf[u][i] = zero;
            if (at < kbytes) {
#pragma unroll
                for (int i = 0; i < PT; ++i) pf[u][i] = *(const u32x4*)(pr[i] + at);
                qf[u] = *(const u32x4*)(qr + at);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u += 2)
#pragma unroll
            for (int i = 0; i < PT; ++i)
                acc[i] = T::mfma(T::make(pf[u][i], pf[u + 1][i]), T::make(qf[u], qf[u + 1]), acc[i]);
    }

#pragma unroll
    for (int i = 0; i < PT; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    // Eight columns of one row per thread: lanes of group g hold columns 4g .. 4g+3 of row
    // lane % 16, so eight columns are two neighbouring groups.
    const int row = threadIdx.x & 15, half = threadIdx.x >> 4, c0 = p0 + half * 8;
    if (half > 1 || row >= a.q_rows || c0 >= a.p_cols) return;
    const float qs = ES == 1 && a.q_scale ? a.q_scale[row] : 1.0f;
    ColumnTerms<T> col[PT];
    Resid8<T> resid;
#pragma unroll
    for (int i = 0; i < PT; ++i) col[i].load(a, c0, a.p_scale ? a.p_scale + (long)i * a.p_cols : nullptr);
    if (a.resid) resid.load(a, row, c0);
    float z[PT][8];
#pragma unroll
    for (int i = 0; i < PT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int l = (half * 2 + h) * 16 + row;
            f32x4 s = sums[0][i][l];
#pragma unroll
            for (int w = 1; w < NW; ++w) s += sums[w][i][l];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[i][4 * h + e] = s[e];
        }
    if constexpr (EPI == EPI_GATED) finish_gated8<T>(a, z[0], z[1], row, c0, qs, col[0], col[1]);
    else finish8<T>(a, z[0], row, c0, qs, col[0], resid);
}

template <class T, int EPI>
void launch(const LinearArgs& a, hipStream_t s) {
    JH_LAUNCH((linear_small_kernel<T, EPI>), dim3((unsigned)(a.p_cols + 15) / 16), dim3(64 * NW), 0, s, a);
    HIP_CHECK(hipGetLastError());
}

template <class T>
void dispatch(const LinearArgs& a, hipStream_t s) {
    if (a.gated) launch<T, EPI_GATED>(a, s);
    else launch<T, EPI_LINEAR>(a, s);
}

}  // namespace

void launch_linear_small(const LinearArgs& a, hipStream_t s) {
    if (a.type == JH_BF16) dispatch<Bf16>(a, s);
    else if (a.type == JH_F16) dispatch<F16>(a, s);
    else if (a.out_f32) dispatch<E4m3Wide>(a, s);
    else dispatch<E4m3>(a, s);
}
