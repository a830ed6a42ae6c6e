// RMS norm with the residual's addition (16-bit or e4m3 output), its gradients, and the
// quantisation of rows to e4m3 with a scale per row.
//
// All are one pass over memory: a row is held in registers, 8 values per chunk and lane,
// between the reduction over it and its use.  Rows of up to 2048 values belong to one
// wavefront (four rows per workgroup), longer ones (up to 16384) to a workgroup of four.
// What bounds them is the memory (a copy of 1 GiB: 5.1 TB/s), on an MI355X:
//
//   rms_norm           9482 x 1024, bf16 + f32 residual -> e4m3     107 MB   23.3 us  4.6 TB/s
//   rms_norm           1 x 768                                                2.2 us  (a launch)
//   quantize_rows      8192 x 8192 f32                              336 MB   62.9 us  5.3 TB/s
//   quantize_rows      9482 x 1152 bf16                              33 MB    9.3 us  3.5 TB/s (1)
//   rms_norm_backward  16384 x 4096 bf16, with dres and dw          537 MB   98.5 us  5.4 TB/s
//   rms_norm_backward  4096 x 16384 bf16, with dres and dw          537 MB    117 us  4.6 TB/s (2)
//   column_sum         512 x 4096, of that dw's parts                 8 MB    4.9 us
//
//   (1) a launch (2 us) and the codes' arithmetic count here: 12.7 us with codes formed in 64 bits
//   (2) one wave per SIMD, so that a row's loads and sums are not under another's; dw's sum included
//
//   forward   s = x + resid, rounded to the residual's type (what is stored is what is
//             normalised); r = 1 / sqrt(mean(s^2) + eps); y = s r w
//   e4m3      p = s w, a = max|p|: the code is the e4m3 value nearest to the exact quotient
//             448 p / a (ties to even), the row's scale r a / 448 (r cancels in the codes)
//   backward  n = s r, g = w dy: ds = r (g - n mean(g n)) (+ dres); dw = sum over rows of dy n
#include <hip/hip_runtime.h>

#include <algorithm>

#include "linear.hpp"

using namespace lin;

namespace {

constexpr int THREADS = 256;
constexpr float E4M3_MAX = 448.0f;

struct F32 {};
template <class T> struct Elem { static constexpr int bytes = 2; };
template <> struct Elem<F32> { static constexpr int bytes = 4; };

// Eight consecutive values in memory, raw (so that loads can be issued before any is used).
template <class T> struct Raw8 { u32x4 v; };
template <> struct Raw8<F32> { f32x4 a, b; };

template <class T>
__device__ inline Raw8<T> load8(const void* base, long i) {
    if constexpr (Elem<T>::bytes == 4) {
        const float* p = (const float*)base + i;
        return {*(const f32x4*)p, *(const f32x4*)(p + 4)};
    } else {
        return {*(const u32x4*)((const uint16_t*)base + i)};
    }
}
template <class T>
__device__ inline void widen(const Raw8<T>& r, float (&v)[8]) {
    if constexpr (Elem<T>::bytes == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = r.a[e];
            v[4 + e] = r.b[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = T::lo(r.v[e]);
            v[2 * e + 1] = T::hi(r.v[e]);
        }
    }
}
template <class T>
__device__ inline void store8(void* base, long i, const float (&v)[8]) {
    if constexpr (Elem<T>::bytes == 4) {
        float* p = (float*)base + i;
        *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        store16<T>((uint16_t*)base + i, v);
    }
}
// v rounded to T and back.
template <class T>
__device__ inline void round_to(float (&v)[8]) {
    if constexpr (Elem<T>::bytes == 2) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t u = T::pack(v[e], v[e + 1]);
            v[e] = T::lo(u);
            v[e + 1] = T::hi(u);
        }
    }
}

__device__ inline float wave_max(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ inline double wave_max(double v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmax(v, __shfl_xor(v, m));
    return v;
}

// Sum or maximum over a row's TPR threads, in every one of them.  With TPR == 256 the four
// waves' values are joined in wave order through `slot` (one per reduction: no barrier is
// needed before its next use within a kernel that reduces once per slot).
template <int TPR>
__device__ inline float row_sum(float v, float* slot) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = ((slot[0] + slot[1]) + slot[2]) + slot[3];
    }
    return v;
}
template <int TPR, class F>
__device__ inline F row_max(F v, F* slot) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = fmax(fmax(slot[0], slot[1]), fmax(slot[2], slot[3]));
    }
    return v;
}

// The e4m3 code of d, |d| <= 448 or NaN, rounded once from 64 bits: the float on the way is
// rounded to odd, which the second rounding cannot mistake for a tie.
__device__ inline uint32_t e4m3_bits(double d0, double d1) {
    auto odd = [](double d) {
        float f = (float)d;
        uint32_t u = __builtin_bit_cast(uint32_t, f);
        const double back = (double)f;
        if (back != d) {
            // f was rounded to nearest: step back to the truncated value, then set the sticky bit
            if (fabs(back) > fabs(d)) u -= 1;
            u |= 1;
        }
        return __builtin_bit_cast(float, u);
    };
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(odd(d0), odd(d1), 0, false) & 0xffffu;
}

// Codes of eight products p = s w (or p = x): the quotient 448 p / a is formed as the
// reciprocal's product with one correction, which makes it the correctly rounded 64-bit
// quotient (448 p is exact in 64 bits; inv is the correctly rounded 1 / a).
__device__ inline u32x2 e4m3_codes(const double (&p)[8], double a, double inv) {
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        double q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double n = 448.0 * p[e + i], q0 = n * inv;
            q[i] = __builtin_fma(__builtin_fma(-q0, a, n), inv, q0);
        }
        h[e >> 1] = e4m3_bits(q[0], q[1]);
    }
    return u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
}

// The same for values of 16 bits, in 32: 448 p has 14 bits at most, so n is exact.  q1 is the
// correctly rounded quotient of n by a (a product with the reciprocal, corrected once), and the
// sign of its remainder, exact too, says on which side of q1 the quotient itself lies.  That
// makes the float rounded to odd.  `lift` (a power of two) keeps the remainder
// normal and n finite where the row's maximum is far from 1.
__device__ inline u32x2 e4m3_codes_half(const float (&p)[8], float a, float inv, float lift) {
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float n = p[e + i] * (E4M3_MAX * lift), q0 = n * inv;
            const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, a, n), inv, q0), r = __builtin_fmaf(-q1, a, n);
            const int u = __builtin_bit_cast(int, q1), away = (__builtin_bit_cast(int, r) ^ u) >> 31;
            // a NaN compares unequal and stays one
            q[i] = __builtin_bit_cast(float, r == 0.0f ? u : (u + away) | 1);
        }
        h[e >> 1] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false) & 0xffffu;
    }
    return u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
}

// One row per TPR threads; NC chunks of 8 values per thread.
template <int TPR>
__device__ inline bool row_of(int rows, long& row, int& lane) {
    row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (THREADS / TPR) + threadIdx.x / TPR;
    lane = threadIdx.x % TPR;
    return row < rows;
}

template <class TX, class TR, int TPR, int NC>
__global__ __launch_bounds__(THREADS) void rms_norm_kernel(RmsNormArgs a) {
    __shared__ float sum_slot[4];
    __shared__ double max_slot[4];
    long row;
    int lane;
    if (!row_of<TPR>(a.rows, row, lane)) return;  // a whole wave, or (TPR 256) a whole workgroup
    float s[NC][8], w[NC][8];
    {
        Raw8<TX> x[NC];
        Raw8<TR> r[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = min((c * TPR + lane) * 8, a.hidden - 8);
            x[c] = load8<TX>(a.x, row * a.ldx + i);
            if (a.resid) r[c] = load8<TR>(a.resid, row * a.ldr + i);
            widen<F32>(Raw8<F32>{*(const f32x4_u*)(a.w + i), *(const f32x4_u*)(a.w + i + 4)}, w[c]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            widen<TX>(x[c], s[c]);
            if (a.resid) {
                float t[8];
                widen<TR>(r[c], t);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[c][e] += t[e];
                round_to<TR>(s[c]);
                if (i < a.hidden) store8<TR>(a.resid_out, row * a.ldro + i, s[c]);
            }
            if (i >= a.hidden) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[c][e] = 0.0f;
            }
        }
    }
    float q = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) q = __builtin_fmaf(s[c][e], s[c][e], q);
    const float r = 1.0f / __builtin_sqrtf(row_sum<TPR>(q, sum_slot) / (float)a.hidden + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = r;
    if (a.out_type == JH_E4M3) {
        double m = 0.0;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmax(m, fabs((double)s[c][e] * (double)w[c][e]));
        m = row_max<TPR>(m, max_slot);
        const double inv = m > 0.0 ? 1.0 / m : 0.0;
        // a row of zeros has scale 0 with eps = 0 too, where r is infinite
        if (lane == 0) a.scales[row] = m > 0.0 || r != r ? (float)(m * (double)r / 448.0) : 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            double p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = (double)s[c][e] * (double)w[c][e];
            if (i < a.hidden) *(u32x2*)((uint8_t*)a.out + row * a.ldo + i) = e4m3_codes(p, m, inv);
        }
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            if (i >= a.hidden) break;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = s[c][e] * r * w[c][e];
            if (a.out_type == JH_BF16) store16<Bf16>((uint16_t*)a.out + row * a.ldo + i, y);
            else store16<F16>((uint16_t*)a.out + row * a.ldo + i, y);
        }
    }
}

template <class TX, int TPR, int NC>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(RmsNormArgs a) {
    __shared__ float max_slot[4];
    long row;
    int lane;
    if (!row_of<TPR>(a.rows, row, lane)) return;
    float v[NC][8];
    {
        Raw8<TX> x[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) x[c] = load8<TX>(a.x, row * a.ldx + min((c * TPR + lane) * 8, a.hidden - 8));
#pragma unroll
        for (int c = 0; c < NC; ++c) widen<TX>(x[c], v[c]);  // a clamped chunk repeats the last: the maximum stays
    }
    float m = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[c][e]));
    m = row_max<TPR>(m, max_slot);
    if (lane == 0) a.scales[row] = m / E4M3_MAX;
    if constexpr (Elem<TX>::bytes == 2) {
        const float lift = m < 0x1p-40f ? 0x1p96f : m > 0x1p100f ? 0x1p-64f : 1.0f;
        const float top = m * lift, inv = m > 0.0f ? 1.0f / top : 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            if (i < a.hidden) *(u32x2*)((uint8_t*)a.out + row * a.ldo + i) = e4m3_codes_half(v[c], top, inv, lift);
        }
        return;
    }
    const double inv = m > 0.0f ? 1.0 / (double)m : 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = (c * TPR + lane) * 8;
        if (i >= a.hidden) break;
        double p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = (double)v[c][e];
        *(u32x2*)((uint8_t*)a.out + row * a.ldo + i) = e4m3_codes(p, (double)m, inv);
    }
}

// Workgroups walk the rows in strides of the grid and keep their part of dw in registers;
// the parts (one per workgroup, so at most 512) are added by column_sum_kernel: no atomics, the
// same sum every time.  TPR 64: the four waves' parts are first joined through LDS, in wave order.
template <class TY, class TS, class TD, int TPR, int NC>
__global__ __launch_bounds__(THREADS) void rms_norm_backward_kernel(RmsNormGradArgs a) {
    constexpr int RPB = THREADS / TPR;
    __shared__ float slot[2][4];
    const int lane = threadIdx.x % TPR;
    float w[NC][8], dw[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = min((c * TPR + lane) * 8, a.hidden - 8);
        widen<F32>(Raw8<F32>{*(const f32x4_u*)(a.w + i), *(const f32x4_u*)(a.w + i + 4)}, w[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[c][e] = 0.0f;
    }
    int turn = 0;
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        Raw8<TY> y[NC];
        Raw8<TS> s[NC];
        Raw8<TD> d[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = min((c * TPR + lane) * 8, a.hidden - 8);
            y[c] = load8<TY>(a.dy, row * a.lddy + i);
            s[c] = load8<TS>(a.s, row * a.lds + i);
            if (a.dres) d[c] = load8<TD>(a.dres, row * a.lddr + i);
        }
        const float r = a.rstd[row];
        float n[NC][8], gy[NC][8], dot = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            widen<TS>(s[c], n[c]);
            widen<TY>(y[c], gy[c]);
            const bool in = (c * TPR + lane) * 8 < a.hidden;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n[c][e] *= r;
                if (a.dw) dw[c][e] = __builtin_fmaf(gy[c][e], n[c][e], dw[c][e]);
                gy[c][e] *= w[c][e];
                dot = in ? __builtin_fmaf(gy[c][e], n[c][e], dot) : dot;
            }
        }
        dot = row_sum<TPR>(dot, slot[turn]) / (float)a.hidden;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            if (i >= a.hidden) break;
            float v[8], t[8];
            if (a.dres) widen<TD>(d[c], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = r * (gy[c][e] - n[c][e] * dot);
                if (a.dres) v[e] += t[e];
            }
            store8<TD>(a.ds, row * a.ldds + i, v);
        }
    }
    if (!a.dw) return;
    float* part = a.partial + (long)blockIdx.x * a.hidden;
    if constexpr (TPR == 64) {
        __shared__ float join[NC][8][64];
        for (int wv = 0; wv < 4; ++wv) {
            if ((int)(threadIdx.x >> 6) == wv) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        join[c][e][lane] = wv ? join[c][e][lane] + dw[c][e] : dw[c][e];
            }
            __syncthreads();
        }
        if (threadIdx.x < 64) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = (c * TPR + lane) * 8;
                if (i >= a.hidden) break;
#pragma unroll
                for (int e = 0; e < 8; ++e) part[i + e] = join[c][e][lane];
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * TPR + lane) * 8;
            if (i >= a.hidden) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) part[i + e] = dw[c][e];
        }
    }
}

// out[c] = sum over r of in[r, c] in FP32: a workgroup owns 64 columns, four per lane of 16,
// and its 64 groups of 16 lanes each add a run of rows, eight loads in flight; the groups' sums
// are added in group order.  Bound by latency: 500 x 1024 takes 4.7 us, of which a launch is 2.
constexpr int SUM_THREADS = 1024, SUM_GROUPS = SUM_THREADS / 16;
__global__ __launch_bounds__(SUM_THREADS) void column_sum_kernel(const float* in, int rows, int cols, float* out) {
    __shared__ __align__(16) float part[SUM_GROUPS][64];
    const int lane = threadIdx.x & 15, grp = threadIdx.x >> 4, c = blockIdx.x * 64 + lane * 4;
    const int per = (rows + SUM_GROUPS - 1) / SUM_GROUPS, r0 = grp * per, r1 = min(rows, r0 + per);
    f32x4 s = {0, 0, 0, 0};
    if (c < cols) {
        for (int r = r0; r < r1; r += 8) {
            f32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *(const f32x4*)(in + (long)min(r + i, r1 - 1) * cols + c);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r + i < r1) s += v[i];
        }
    }
    *(f32x4*)&part[grp][lane * 4] = s;
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < cols) {
        float t = 0.0f;
#pragma unroll
        for (int g = 0; g < SUM_GROUPS; ++g) t += part[g][threadIdx.x];
        out[blockIdx.x * 64 + threadIdx.x] = t;
    }
}

// f<TPR, NC>() for the number of 8-value chunks each of a row's threads holds.
template <class F>
void dispatch_row(int hidden, F&& f) {
    const int chunks = hidden / 8;
    if (chunks <= 256) {
        switch ((chunks + 63) / 64) {
            case 1: f.template operator()<64, 1>(); break;
            case 2: f.template operator()<64, 2>(); break;
            case 3: f.template operator()<64, 3>(); break;
            default: f.template operator()<64, 4>(); break;
        }
    } else {
        switch ((chunks + 255) / 256) {
            case 2: f.template operator()<256, 2>(); break;
            case 3: f.template operator()<256, 3>(); break;
            case 4: f.template operator()<256, 4>(); break;
            case 5:
            case 6: f.template operator()<256, 6>(); break;
            default: f.template operator()<256, 8>(); break;
        }
    }
}

int row_blocks(int rows, int tpr) {
    const int per = THREADS / tpr;
    return rows / per + (rows % per != 0);
}
// A launch holds fewer than 2^32 threads along x: more rows than 2^20 workgroups have go along y.
dim3 row_grid(int rows, int tpr) {
    const int b = row_blocks(rows, tpr), x = std::min(b, 1 << 20);
    return dim3((unsigned)x, (unsigned)((b - 1) / x + 1));
}

template <class TX, class TR>
void launch_norm(const RmsNormArgs& a, hipStream_t s) {
    dispatch_row(a.hidden, [&]<int TPR, int NC>() {
        JH_LAUNCH((rms_norm_kernel<TX, TR, TPR, NC>), row_grid(a.rows, TPR), dim3(THREADS), 0, s, a);
    });
}
template <class TY, class TS, class TD>
void launch_norm_backward(const RmsNormGradArgs& a, hipStream_t s) {
    dispatch_row(a.hidden, [&]<int TPR, int NC>() {
        JH_LAUNCH((rms_norm_backward_kernel<TY, TS, TD, TPR, NC>), dim3((unsigned)a.blocks), dim3(THREADS), 0, s, a);
    });
}
template <class TY>
void launch_norm_backward_of(const RmsNormGradArgs& a, hipStream_t s) {
    const bool s32 = a.s_type == JH_F32, d32 = a.ds_type == JH_F32;
    if (s32 && d32) launch_norm_backward<TY, F32, F32>(a, s);
    else if (s32) launch_norm_backward<TY, F32, TY>(a, s);
    else if (d32) launch_norm_backward<TY, TY, F32>(a, s);
    else launch_norm_backward<TY, TY, TY>(a, s);
}

constexpr int MAX_HIDDEN = 16384;

[[noreturn]] void refuse(const char* op, const char* what) {
    throw jh_error(JH_ERR_INVALID, std::string(op) + ": " + what);
}

void check_width(const char* op, int hidden) {
    if (hidden <= 0 || hidden % 8 || hidden > MAX_HIDDEN) refuse(op, "row length must be a multiple of 8, at most 16384");
}

bool plain_type(int t) { return t == JH_F32 || t == JH_BF16 || t == JH_F16; }

// e4m3 rows are written 8 bytes at a time.
void check_codes(const char* op, const void* q, size_t ld, size_t rows, size_t cols) {
    if (!q) refuse(op, "the e4m3 output is null");
    if (((uintptr_t)q | (rows > 1 ? ld : 0)) & 7) refuse(op, "e4m3 rows are not 8-byte aligned");
    if (rows > 1 && ld < cols) refuse(op, "the e4m3 output: row stride below its columns");
    if (ld > ((size_t)1 << 22)) refuse(op, "the e4m3 output: row stride over 4 MiB");
}

// Workgroups of the backward pass, each with a part of dw: as many as the GPU holds at once, fewer where
// there are fewer rows than they take.  That is two per CU of up to 8192 columns, one of more, whose
// six or eight chunks per thread need over 256 registers.  (One and two per CU, bf16 with dres and dw:
// 16384 x 4096 111 and 104 us, 8192 x 8192 108 and 108, 5461 x 12288 111 and 117, 4096 x 16384 117
// and 127, 300 x 16384 22 and 26.)
int backward_blocks(int rows, int hidden) {
    return std::max(1, std::min(row_blocks(rows, hidden <= 2048 ? 64 : 256), hidden <= 8192 ? 512 : 256));
}

}  // namespace

void rms_norm(const RmsNormArgs& args, hipStream_t s) {
    RmsNormArgs a = args;
    const char* op = "rms_norm";
    check_width(op, a.hidden);
    if (!plain_type(a.x_type)) refuse(op, "x must be f32, bf16 or f16");
    if (a.resid_type != JH_F32 && a.resid_type != a.x_type) refuse(op, "the residual has x's type or f32");
    if (a.out_type != JH_E4M3 && a.out_type != (a.x_type == JH_F32 && a.out_type == JH_F16 ? JH_F16 : a.x_type == JH_F32 ? JH_BF16 : a.x_type))
        refuse(op, "the output is e4m3 or x's 16-bit type (either one for f32)");
    if (!(a.eps >= 0.0f)) refuse(op, "eps must not be negative");
    if ((a.resid == nullptr) != (a.resid_out == nullptr)) refuse(op, "resid and resid_out go together");
    if (a.rows == 0) return;
    const size_t rows = a.rows, h = a.hidden;
    for (long* ld : {&a.ldx, &a.ldr, &a.ldro, &a.ldo}) *ld = row_stride(*ld, rows, h);
    if (!a.w) refuse(op, "w is null");
    check_matrix(op, "x", a.x, a.ldx, rows, h, a.x_type);
    if (a.resid) {
        check_matrix(op, "resid", a.resid, a.ldr, rows, h, a.resid_type);
        check_matrix(op, "resid_out", a.resid_out, a.ldro, rows, h, a.resid_type);
    }
    if (a.out_type == JH_E4M3) {
        check_codes(op, a.out, a.ldo, rows, h);
        if (!a.scales) refuse(op, "e4m3 output needs scales");
    } else {
        check_matrix(op, "out", a.out, a.ldo, rows, h, a.out_type);
        if (a.scales) refuse(op, "scales belong to e4m3 output");
    }
    const Span in[3] = {span_of(a.x, a.ldx, rows, h, a.x_type), vector_span(a.w, h),
                        span_of(a.resid, a.ldr, rows, h, a.resid_type)};
    const Span out[4] = {span_of(a.out, a.ldo, rows, h, a.out_type), vector_span(a.scales, rows), vector_span(a.rstd, rows),
                         span_of(a.resid_out, a.ldro, rows, h, a.resid_type)};
    const bool in_place = a.resid_out == a.resid && a.ldro == a.ldr;
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 3; ++i)
            if (!(o == 3 && i == 2 && in_place)) check_disjoint(op, "an output", out[o], "an input", in[i]);
        for (int i = 0; i < o; ++i) check_disjoint(op, "an output", out[o], "another", out[i]);
    }
    if (a.x_type == JH_F32) launch_norm<F32, F32>(a, s);
    else if (a.x_type == JH_BF16 && a.resid_type == JH_F32) launch_norm<Bf16, F32>(a, s);
    else if (a.x_type == JH_BF16) launch_norm<Bf16, Bf16>(a, s);
    else if (a.resid_type == JH_F32) launch_norm<F16, F32>(a, s);
    else launch_norm<F16, F16>(a, s);
    HIP_CHECK(hipGetLastError());
}

void quantize_rows(const RmsNormArgs& args, hipStream_t s) {
    RmsNormArgs a = args;
    const char* op = "quantize_rows";
    check_width(op, a.hidden);
    if (!plain_type(a.x_type)) refuse(op, "x must be f32, bf16 or f16");
    if (a.rows == 0) return;
    const size_t rows = a.rows, h = a.hidden;
    for (long* ld : {&a.ldx, &a.ldo}) *ld = row_stride(*ld, rows, h);
    check_matrix(op, "x", a.x, a.ldx, rows, h, a.x_type);
    check_codes(op, a.out, a.ldo, rows, h);
    if (!a.scales) refuse(op, "scales is null");
    const Span x = span_of(a.x, a.ldx, rows, h, a.x_type), q = span_of(a.out, a.ldo, rows, h, JH_E4M3);
    const Span sc = vector_span(a.scales, rows);
    check_disjoint(op, "q", q, "x", x);
    check_disjoint(op, "scales", sc, "x", x);
    check_disjoint(op, "scales", sc, "q", q);
    dispatch_row(a.hidden, [&]<int TPR, int NC>() {
        const dim3 grid = row_grid(a.rows, TPR);
        if (a.x_type == JH_F32) JH_LAUNCH((quantize_rows_kernel<F32, TPR, NC>), grid, dim3(THREADS), 0, s, a);
        else if (a.x_type == JH_BF16) JH_LAUNCH((quantize_rows_kernel<Bf16, TPR, NC>), grid, dim3(THREADS), 0, s, a);
        else JH_LAUNCH((quantize_rows_kernel<F16, TPR, NC>), grid, dim3(THREADS), 0, s, a);
    });
    HIP_CHECK(hipGetLastError());
}

size_t rms_norm_backward_workspace(int rows, int hidden) {
    check_width("rms_norm_backward", hidden);
    return (size_t)backward_blocks(rows, hidden) * hidden * 4;
}

void rms_norm_backward(const RmsNormGradArgs& args, size_t workspace_bytes, hipStream_t s) {
    const char* op = "rms_norm_backward";
    RmsNormGradArgs a = args;
    check_width(op, a.hidden);
    if (!plain_type(a.dy_type)) refuse(op, "dy must be f32, bf16 or f16");
    if ((a.s_type != JH_F32 && a.s_type != a.dy_type) || (a.ds_type != JH_F32 && a.ds_type != a.dy_type))
        refuse(op, "s and ds have dy's type or f32");
    const size_t rows = a.rows, h = a.hidden, need = rms_norm_backward_workspace(a.rows, a.hidden);
    if (a.dw && !a.w) refuse(op, "w is null");  // read whatever the number of rows
    for (long* ld : {&a.lddy, &a.lds, &a.lddr, &a.ldds}) *ld = row_stride(*ld, rows, h);
    if (a.dw && (!a.partial || ((uintptr_t)a.partial & 15))) refuse(op, "dw needs a 16-byte aligned workspace");
    if (a.dw && workspace_bytes < need) refuse(op, "workspace too small");
    if (rows) {
        if (!a.w || !a.rstd) refuse(op, "w and rstd are needed");
        check_matrix(op, "dy", a.dy, a.lddy, rows, h, a.dy_type);
        check_matrix(op, "s", a.s, a.lds, rows, h, a.s_type);
        if (a.dres) check_matrix(op, "dres", a.dres, a.lddr, rows, h, a.ds_type);
        check_matrix(op, "ds", a.ds, a.ldds, rows, h, a.ds_type);
    } else if (!a.dw) {
        return;
    }
    // ds may take the place of dres, dy or s: a row is read whole before it is written.
    const Span ds = span_of(a.ds, a.ldds, rows, h, a.ds_type);
    const struct {
        const void* p;
        long ld;
        int type;
    } in[3] = {{a.dy, a.lddy, a.dy_type}, {a.s, a.lds, a.s_type}, {a.dres, a.lddr, a.ds_type}};
    const Span dw = vector_span(a.dw, h), ws = span_of(a.dw ? a.partial : nullptr, need, 1, need, JH_E4M3);
    for (const auto& i : in) {
        const Span sp = span_of(i.p, i.ld, rows, h, i.type);
        if (!(i.p == a.ds && i.ld == a.ldds && i.type == a.ds_type)) check_disjoint(op, "ds", ds, "an input", sp);
        check_disjoint(op, "dw", dw, "an input", sp);
        check_disjoint(op, "the workspace", ws, "an input", sp);
    }
    for (const float* v : {a.w, a.rstd}) {
        const Span sp = vector_span(v, v == a.w ? h : rows);
        check_disjoint(op, "ds", ds, "an input", sp);
        check_disjoint(op, "dw", dw, "an input", sp);
        check_disjoint(op, "the workspace", ws, "an input", sp);
    }
    check_disjoint(op, "dw", dw, "ds", ds);
    check_disjoint(op, "dw", dw, "the workspace", ws);
    check_disjoint(op, "ds", ds, "the workspace", ws);

    a.blocks = backward_blocks(a.rows, a.hidden);
    if (a.dy_type == JH_F32) launch_norm_backward<F32, F32, F32>(a, s);
    else if (a.dy_type == JH_BF16) launch_norm_backward_of<Bf16>(a, s);
    else launch_norm_backward_of<F16>(a, s);
    HIP_CHECK(hipGetLastError());
    if (a.dw) launch_column_sum(a.partial, a.blocks, a.hidden, a.dw, s);
}

void launch_column_sum(const float* in, int rows, int cols, float* out, hipStream_t s) {
    JH_LAUNCH(column_sum_kernel, dim3((unsigned)(cols + 63) / 64), dim3(SUM_THREADS), 0, s, in, rows, cols, out);
    HIP_CHECK(hipGetLastError());
}
