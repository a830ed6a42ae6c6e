// Linear layers and gated projections: checks, the choice of kernel, the element-wise half of
// their backward passes and the sums over splits of a contraction.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "linear.hpp"

using namespace lin;

namespace {

constexpr int THREADS = 256;

// act'(z) and act(z) together.
__device__ inline void act_and_grad(float z, int act, float& value, float& grad) {
    if (act == JH_ACT_NONE) {
        value = z;
        grad = 1.0f;
    } else if (act == JH_ACT_RELU) {
        value = z < 0.0f ? 0.0f : z;
        grad = z > 0.0f ? 1.0f : 0.0f;
        if (z != z) grad = z;
    } else if (act == JH_ACT_GELU) {
        float a, e;
        const float q = normal_tail(z, a, e), pdf = 0.3989422804014327f * e;
        value = gelu_of(z, a, q);
        grad = __builtin_fmaf(z, pdf, z < 0.0f ? q : 1.0f - q);
    } else {
        const float a = act == JH_ACT_SILU ? 1.0f : kTanhA, b = act == JH_ACT_SILU ? 0.0f : kTanhA * kTanhB;
        // z^2 short of infinity, whose products with 0 (b, or 1 - s) would be NaN
        const float zz = fminf(z * z, 1e30f), s = sigmoid(z * __builtin_fmaf(b, zz, a));
        value = z * s;
        grad = __builtin_fmaf(value * (1.0f - s), __builtin_fmaf(3.0f * b, zz, a), s);
    }
}

template <class T>
__device__ inline void load8_of(const void* p, float (&v)[8]) {
    const u32x4 r = *(const u32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = T::lo(r[e]);
        v[2 * e + 1] = T::hi(r[e]);
    }
}

// dz = dy act'(pre) (rounded to T) and the column sums of its unrounded values, a part per
// blockIdx.y.  A lane owns 8 columns, the four waves of a workgroup every fourth of its rows;
// their sums are joined in wave order.  dz is kept because both products read it, one of them by
// columns, and rounded because the matrix instruction takes 16 bits: dx and dw are off by 0.0023
// of their norm so (9482 x 1024 x 4096 bf16, against 64 bits), by 0.0017 for their own rounding
// alone.  Bound by memory: 9482 x 1024 bf16 gelu, 58 MB, takes 18 to 20 us (3.1 TB/s; 3 more
// with four rows in flight per wave).
template <class T>
__global__ __launch_bounds__(THREADS) void act_grad_kernel(ActGradArgs a) {
    __shared__ float join[4][64][9];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long c = ((long)blockIdx.x * 64 + lane) * 8;
    const long r0 = (long)blockIdx.y * a.rows_per_block, r1 = min((long)a.rows, r0 + a.rows_per_block);
    float sum[8] = {};
    if (c < a.n) {
        for (long r = r0 + wave; r < r1; r += 4) {
            float dz[8];
            load8_of<T>((const uint16_t*)a.dy + r * a.lddy + c, dz);
            if (a.pre) {
                float z[8];
                load8_of<T>((const uint16_t*)a.pre + r * a.ldpre + c, z);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float v, d;
                    act_and_grad(z[e], a.act, v, d);
                    dz[e] *= d;
                }
                store16<T>((uint16_t*)a.dz + r * a.n + c, dz);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += dz[e];
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) join[wave][lane][e] = sum[e];
    __syncthreads();
    if (wave == 0 && c < a.n) {
        float* o = a.partial + (long)blockIdx.y * a.n + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = ((join[0][lane][e] + join[1][lane][e]) + join[2][lane][e]) + join[3][lane][e];
    }
}

// [dg du] = [dh u act'(g), dh act(g)], rounded to T as dz is.  Bound by memory: 9482 x 1152 bf16, 109 MB,
// takes 20 us (5.5 TB/s).
template <class T>
__global__ __launch_bounds__(THREADS) void gated_grad_kernel(GatedGradArgs a) {
    const long per = a.inter / 8, i = (long)blockIdx.x * THREADS + threadIdx.x;
    const long r = i / per, c = (i - r * per) * 8;
    if (r >= a.rows) return;
    float dh[8], g[8], u[8], dg[8], du[8];
    load8_of<T>((const uint16_t*)a.dh + r * a.lddh + c, dh);
    load8_of<T>((const uint16_t*)a.gu + r * a.ldgu + c, g);
    load8_of<T>((const uint16_t*)a.gu + r * a.ldgu + a.inter + c, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v, d;
        act_and_grad(g[e], a.act, v, d);
        dg[e] = dh[e] * u[e] * d;
        du[e] = dh[e] * v;
    }
    uint16_t* o = (uint16_t*)a.dgu + r * 2 * a.inter + c;
    store16<T>(o, dg);
    store16<T>(o + a.inter, du);
}

// out[r, c] = sum over s of partial[s][r, c], in split order.  Bound by memory: four parts of
// 2304 x 768, 32 MB, take 6.2 us (5.1 TB/s), eight, 60 MB, 10 us (6 TB/s, partly from cache).
template <class T>
__global__ __launch_bounds__(THREADS) void split_sum_kernel(const float* partial, int splits, int rows, int cols,
                                                            void* out, long ldo, int out_f32) {
    const long per = cols / 8, i = (long)blockIdx.x * THREADS + threadIdx.x;
    const long r = i / per, c = (i - r * per) * 8;
    if (r >= rows) return;
    const long plane = (long)rows * cols;
    const float* p = partial + r * cols + c;
    f32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    for (int s0 = 0; s0 < splits; s0 += 4) {  // four planes in flight; those past the last are read again, not added
        f32x4 v[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[i][h] = *(const f32x4*)(p + min(s0 + i, splits - 1) * plane + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i < splits) {
                lo += v[i][0];
                hi += v[i][1];
            }
        }
    }
    if (out_f32) {
        float* o = (float*)out + r * ldo + c;
        *(f32x4*)o = lo;
        *(f32x4*)(o + 4) = hi;
    } else {
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        store16<T>((uint16_t*)out + r * ldo + c, v);
    }
}

unsigned blocks_of(long items, const char* what) {
    const long b = (items + THREADS - 1) / THREADS;
    if (b * THREADS >= 1L << 32) throw jh_error(JH_ERR_INVALID, std::string(what) + ": too many elements");
    return (unsigned)b;
}

long round_up(long v, long to) { return (v + to - 1) / to * to; }

// ---------------------------------------------------------------- choice of kernel

long steps_of(const LinearArgs& a) {
    const long es = a.type == JH_E4M3 ? 1 : 2;
    return (a.k * es + STEP_BYTES - 1L) / STEP_BYTES;
}
long tiles_of(const LinearArgs& a, int p, int q) {
    const long cols = a.gated ? 2L * a.p_cols : a.p_cols;
    return ((cols + p - 1) / p) * ((a.q_rows + q - 1L) / q);
}

// What a launch of each kernel takes, in us, from its number of tiles and of K steps: a start
// and an end per round of tiles (launch, first loads, epilogue) and a time per step that grows
// with the CUs at work (shared L2 and power).  The constants are fits to times on an MI355X (256 CUs):
// forward products to 42 sizes whose inputs, in three sets, take turns, as a layer meets its own (the
// kernel that comes out cheapest takes 0.1 % longer than the fastest in the mean, 6 % at worst; on 110
// other sizes, inputs out of cache and whole rounds of 256 x 256 tiles among the choices, 1.7 % and 25 %);
// gradients to 124 sizes, log-uniform ones and training widths, with as many sets of inputs as 700 MB
// hold, so that none is left in the 256 MB of cache, but dz just written, as the activation's gradient
// leaves it (0.6 % and 11 %; on 140 other sizes 1.1 % and 18 %).  Some of them, bf16, gradients in
// their best number of parts (us, the kernel taken in brackets):
//
//   rows x n x k              Small   Deep    Pair    Tall    256 x 256
//   512 x 768 x 768           [7.0]   9.9     12.2    13.8    21.2
//   1024 x 1024 x 4096        [19.9]  30.4    51.3    45.1    70.7
//   1024 x 4096 x 1024        19.5    [14.3]  19.4    18.4    26.2
//   9482 x 768 x 1152         32.3    27.1    25.4    [21.8]  29.6
//   2048 x 4096 x 4096        111     71.6    68.6    [59.9]  74.9
//   4096 x 4096 x 4096        204     143     135     121     [101]
//   9482 x 4096 x 1024        147     111     99.8    96.6    [88.3]
//   dx of 4096 x 1024 x 768   18.6    [15.5]  18.8            27.2
//   dx of 9482 x 2304 x 768   65.9    48.9    [42.5]          49.9
//   dx of 9482 x 1152 x 4096  178     143     107             [102]
//   dw of 1024 x 4096 x 1024  23.3    [16.3]  19.3            31.1
//   dw of 4096 x 4096 x 1024  70.6    [45.1]  48.2            53.6
//   dw of 8192 x 1152 x 2048  92.9    75.0    [58.9]          61.3
//   dw of 9482 x 2304 x 768   73.8    58.7    51.8            [54.6]
//   dw of 16384 x 2304 x 1024 162     122     96.4            [90.3]
//   dw of 8192 x 4096 x 8192  1024    637     535             [461]
//
// (64 x 64 tiles of which four groups of waves shared the contraction were the fastest in none of 240
// sizes: 18.2 us for dw of 1024 x 768 x 2048, Small 13.0.)
enum { SMALL = JH_KERNEL_SMALL, DEEP = JH_KERNEL_DEEP, PAIR = JH_KERNEL_PAIR, TALL = JH_KERNEL_TALL,
       WIDE = JH_KERNEL_WIDE, KERNELS };
constexpr long CUS = 256;

double cost(int kernel, const LinearArgs& a, long splits) {
    const double s = (double)((steps_of(a) + splits - 1) / splits);
    const bool by_cols = a.layout != ROWS_ROWS, both = a.layout == COLS_COLS;
    // `of(n)`: a round of n tiles, `slots` of which the GPU holds
    auto rounds = [](long t, long slots, auto of) {
        return (double)(t / slots) * of((double)slots) + (t % slots ? of((double)(t % slots)) : 0.0);
    };
    auto load = [](double t) { return std::min(1.0, t / (double)CUS); };
    switch (kernel) {
        case SMALL: {
            const long t = tiles_of(a, 64, 64) * splits;
            if (by_cols && t <= CUS) return 3.9 + 0.36 * s;
            if (by_cols) return rounds(t, 2 * CUS, [&](double) { return (both ? 0.5 : 0.47) * s + 1.6; }) + 4.1;
            if (t <= CUS) return 3.7 + (0.215 + 0.05 * load((double)t)) * s;
            return rounds(t, 2 * CUS, [&](double) { return 0.42 * s + 2.0; }) + 1.0;
        }
        case DEEP: {
            const long t = tiles_of(a, 128, 128) * splits;
            if (by_cols) return rounds(t, CUS, [&](double) { return (both ? 0.63 : 0.61) * s + 4.1; }) + 3.2;
            return rounds(t, CUS, [&](double n) { return s * (0.35 + 0.19 * load(n)) + 3.0; }) + 1.5;
        }
        case PAIR: {
            const long t = tiles_of(a, 128, 128) * splits;
            if (by_cols) {
                const double full = both ? 1.03 : 1.05, alone = both ? 0.75 : 0.7;
                return rounds(t, 2 * CUS, [&](double n) { return s * (n > CUS ? full : alone + 0.16 * load(n)) + 4.9; }) + 1.8;
            }
            return rounds(t, 2 * CUS, [&](double n) { return s * (n > CUS ? 0.92 : 0.62 + 0.16 * load(n)) + 5.0; }) + 1.0;
        }
        case TALL: {
            const long t = tiles_of(a, 128, 256) * splits;
            return rounds(t, CUS, [&](double n) { return s * (0.54 + 0.33 * load(n)) + 4.2; }) + 2.5;
        }
        default: {
            const long t = tiles_of(a, 256, 256) * splits;
            const double alone = both ? 1.28 : by_cols ? 1.04 : 0.88, all = both ? 1.62 : by_cols ? 1.51 : 1.37;
            return rounds(t, CUS, [&](double n) { return s * (alone + (all - alone) * load(n) * load(n)) + (by_cols ? 11.1 : 9.0); }) +
                   (by_cols ? 0.0 : 1.0);
        }
    }
}

// Whether a launch can hold the kernel's tiles along x, where it has fewer than 2^32 threads.  (2^30 rows
// by 8 columns: 2^24 tiles of 64 x 64 by 256 threads are too many, 2^23 of 128 x 128 are not.)
bool launches(int kernel, const LinearArgs& a) {
    const int side = kernel == WIDE ? 256 : kernel == SMALL ? 64 : 128;
    const long threads = kernel == SMALL || kernel == PAIR ? 256 : 512;
    return tiles_of(a, side, kernel == TALL ? 256 : side) * threads < 1L << 32;
}

struct Choice {
    int kernel;  // KERNELS: none can be launched
    int splits;
    double cost;
};

// The cheapest kernel and, for gradients, number of parts of the contraction, whose FP32 sums
// take `splits` outputs' worth of memory (at most 16; 48 MiB of rows' gradients, 192 MiB of
// weights') and one more kernel.
constexpr long MAX_SPLITS = 16, MIN_STEPS = 4;
long split_bytes(const LinearArgs& a) { return (a.layout == COLS_COLS ? 192L : 48L) << 20; }
Choice pick(const LinearArgs& a, bool gradient) {
    Choice best{KERNELS, 1, 1e30};
    const double out = (double)a.q_rows * a.p_cols * 4;
    for (long splits = 1; splits <= (gradient ? MAX_SPLITS : 1); splits += splits < 4 ? 1 : splits < 8 ? 2 : 4) {
        if (splits > 1 && (steps_of(a) < splits * MIN_STEPS || out * splits > split_bytes(a))) break;
        const double sum = splits > 1 ? 3.7 + (2 * splits + 0.5) * out / 9.9e6 : 0.0;  // written and read, mostly in cache
        for (int kernel = 0; kernel < KERNELS; ++kernel) {
            // no room there for e4m3 fragments widened to bf16; Tall gains nothing by columns (9482 x 768
            // x 2304: 38.2 us, Pair 37.5)
            if (kernel >= TALL && a.type == JH_E4M3 && a.out_f32) continue;
            if (kernel == TALL && a.layout != ROWS_ROWS) continue;
            if (!launches(kernel, a)) continue;
            const double c = cost(kernel, a, splits) + sum;
            if (c < best.cost) best = {kernel, (int)splits, c};
        }
    }
    return best;
}

// Output rows [r0, r0 + rows) of a product.
LinearArgs row_range(const LinearArgs& a, int r0, int rows) {
    LinearArgs r = a;
    const long es = a.type == JH_E4M3 ? 1 : 2, os = a.out_f32 ? 4 : 2;
    r.q = (const uint8_t*)a.q + (a.layout == COLS_COLS ? r0 : r0 * a.ldq) * es;
    r.q_rows = rows;
    if (a.q_scale) r.q_scale = a.q_scale + r0;
    if (a.resid) r.resid = (const uint8_t*)a.resid + r0 * a.ldr * os;
    r.out = (uint8_t*)a.out + r0 * a.ldo * os;
    if (a.pre) r.pre = (uint8_t*)a.pre + r0 * a.ldpre * 2;
    return r;
}

// Rows that 256 x 256 tiles take in whole rounds of the CUs, where that and another kernel
// for the rest come cheaper than any kernel alone; else 0.  18000 x 1024 x 4096 (284 tiles): 164
// us at once, 127 as 16384 rows and 1616 on 64 x 64 tiles; 5000 x 4096 x 4096: 161 and 138.  The
// second launch and the drain between cost 3 us, so that a last round half full stays where it is
// (9482 x 2304 x 768: 46.5 us, in two 48.4).
int whole_rounds(const LinearArgs& a, double alone) {
    if (a.type == JH_E4M3 && a.out_f32) return 0;
    const long across = tiles_of(row_range(a, 0, 1), 256, 256), rounds = tiles_of(a, 256, 256) / CUS;
    const long rows = rounds * CUS / across * 256;
    if (rows <= 0 || rows >= a.q_rows || !launches(WIDE, row_range(a, 0, (int)rows))) return 0;
    const double c = cost(WIDE, row_range(a, 0, (int)rows), 1) +
                     pick(row_range(a, (int)rows, a.q_rows - (int)rows), false).cost + 3.0;
    return c < alone ? (int)rows : 0;
}

// What a product runs on, settled before anything is launched: one kernel, or 256 x 256 tiles for its
// first `whole` rows and another kernel for the rest.
struct Plan {
    int kernel, splits, whole, rest;
};

// Up to 16 rows, W streams past them from memory (16 x 4096 x 4096: 10.1 us, 16.5 on 64 x 64
// tiles; 17 to 32 rows, two blocks of them, took 18.2 against 17.6).
constexpr int STREAM_ROWS = 16;

Plan plan(const char* op, const LinearArgs& a, bool gradient) {
    if (!gradient && a.q_rows <= STREAM_ROWS) return {JH_KERNEL_STREAM, 1, 0, 0};
    const Choice c = pick(a, gradient);
    if (c.kernel == KERNELS) throw jh_error(JH_ERR_INVALID, std::string(op) + ": too large");
    Plan p{c.kernel, c.splits, c.splits == 1 ? whole_rounds(a, c.cost) : 0, 0};
    if (p.whole) {
        p.kernel = WIDE;
        p.rest = pick(row_range(a, p.whole, a.q_rows - p.whole), false).kernel;
    }
    return p;
}

long partial_bytes(const LinearArgs& a, const Plan& p) {
    return p.splits > 1 ? round_up((long)p.splits * a.q_rows * a.p_cols * 4, 256) : 0;
}

void launch(int kernel, const LinearArgs& a, hipStream_t s) {
    if (kernel == JH_KERNEL_STREAM) launch_linear_small(a, s);
    else if (kernel == WIDE) launch_linear_wide(a, s);
    else launch_linear_tile(a, kernel == SMALL ? LinearTile::Small : kernel == DEEP ? LinearTile::Deep
                               : kernel == PAIR ? LinearTile::Pair : LinearTile::Tall, s);
}

template <class T>
void split_sum(const LinearArgs& a, hipStream_t s) {
    const unsigned b = blocks_of((long)a.q_rows * (a.p_cols / 8), "linear");
    JH_LAUNCH(split_sum_kernel<T>, dim3(b), dim3(THREADS), 0, s, a.partial, a.splits, a.q_rows, a.p_cols, a.out, a.ldo,
              a.out_f32);
    HIP_CHECK(hipGetLastError());
}

// A product by its plan; the parts of a contraction that is split go to `partial`.
void run(LinearArgs a, const Plan& p, float* partial, hipStream_t s) {
    a.splits = p.splits;
    a.split_steps = p.splits > 1 ? (int)((steps_of(a) + p.splits - 1) / p.splits) : 0x7fffffff;
    a.partial = p.splits > 1 ? partial : nullptr;
    if (p.whole) {
        launch(p.kernel, row_range(a, 0, p.whole), s);
        return launch(p.rest, row_range(a, p.whole, a.q_rows - p.whole), s);
    }
    launch(p.kernel, a, s);
    if (p.splits == 1) return;
    if (a.type == JH_BF16) split_sum<Bf16>(a, s);
    else split_sum<F16>(a, s);
}

// ---------------------------------------------------------------- checks

[[noreturn]] void refuse(const char* op, const char* what) {
    throw jh_error(JH_ERR_INVALID, std::string(op) + ": " + what);
}

int type_bytes(int type) { return type == JH_F32 ? 4 : type == JH_E4M3 ? 1 : 2; }

}  // namespace

// ---------------------------------------------------------------- shared argument checks

void check_matrix(const char* op, const char* name, const void* p, size_t ld, size_t rows, size_t cols, int type) {
    const size_t bytes = type_bytes(type);
    const char* what = !p                                          ? " is null"
                       : (uintptr_t)p & 15                         ? " is not 16-byte aligned"
                       : rows <= 1                                 ? nullptr
                       : ld < cols                                 ? ": row stride below its columns"
                       : ld > ((size_t)1 << 22) / bytes            ? ": row stride over 4 MiB"
                       : ld * bytes % 16                           ? ": rows are not 16-byte aligned"
                                                                   : nullptr;
    if (!what && cols * bytes > ((size_t)1 << 22)) what = ": rows over 4 MiB";
    if (what) throw jh_error(JH_ERR_INVALID, std::string(op) + ": " + name + what);
}

Span span_of(const void* p, size_t ld, size_t rows, size_t cols, int type) {
    return Span{(uintptr_t)p, p ? rows : 0, cols * type_bytes(type), std::max(ld, cols) * type_bytes(type)};
}

Span vector_span(const float* p, size_t n) { return span_of(p, n, p ? 1 : 0, n, JH_F32); }

// Whether two strided matrices share a byte.  With equal row strides their columns are
// compared within a row (two column ranges of one buffer do not overlap); otherwise their
// whole extents are.
bool spans_overlap(const Span& a, const Span& b) {
    if (!a.rows || !b.rows || !a.width || !b.width) return false;
    const uintptr_t a1 = a.at + (a.rows - 1) * a.stride + a.width, b1 = b.at + (b.rows - 1) * b.stride + b.width;
    if (a1 <= b.at || b1 <= a.at) return false;
    if (a.stride != b.stride || a.rows == 1 || b.rows == 1) return true;
    const uintptr_t d = (b.at > a.at ? b.at - a.at : a.stride - (a.at - b.at) % a.stride) % a.stride;
    return d < a.width || d + b.width > a.stride;
}

void check_disjoint(const char* op, const char* out_name, const Span& out, const char* in_name, const Span& in) {
    if (spans_overlap(out, in))
        throw jh_error(JH_ERR_INVALID, std::string(op) + ": " + out_name + " overlaps " + in_name);
}

// ---------------------------------------------------------------- entry points

namespace {

void check_sizes(const char* op, int type, size_t rows, size_t n, size_t k) {
    if (type != JH_BF16 && type != JH_F16 && type != JH_E4M3) refuse(op, "type must be bf16, f16 or e4m3");
    if (n == 0 || k == 0) refuse(op, "empty feature dimension");
    if (n % 8) refuse(op, "output features must be a multiple of 8");
    if (k % (type == JH_E4M3 ? 16 : 8)) refuse(op, "input features must be a multiple of 16 bytes");
    if (rows > ((size_t)1 << 30) || n > ((size_t)1 << 22)) refuse(op, "too large");
}

void check_act(const char* op, int act) {
    if (act < JH_ACT_NONE || act > JH_ACT_SILU) refuse(op, "unknown activation");
}

}  // namespace

void linear_forward(const LinearArgs& args, size_t rows, size_t n, size_t k, int out_type, hipStream_t s) {
    LinearArgs a = args;
    const char* op = a.gated ? "gated_ffn" : "linear";
    check_sizes(op, a.type, rows, n, k);
    check_act(op, a.act);
    const int half = a.type == JH_E4M3 ? JH_BF16 : a.type;
    if (out_type != half && (a.gated || out_type != JH_F32))
        refuse(op, a.gated ? "the output has the operands' type (bf16 for e4m3)"
                           : "the output has the operands' type (bf16 for e4m3) or f32");
    if (a.type != JH_E4M3 && (a.p_scale || a.q_scale)) refuse(op, "scales belong to e4m3 operands");
    if (a.type == JH_E4M3 && a.pre) refuse(op, "pre-activations are kept for 16-bit operands");
    const size_t w_rows = a.gated ? 2 * n : n;
    if (rows == 0) return;
    a.ldq = row_stride(a.ldq, rows, k);
    a.ldo = row_stride(a.ldo, rows, n);
    a.ldr = row_stride(a.ldr, rows, n);
    a.ldpre = row_stride(a.ldpre, rows, w_rows);
    check_matrix(op, "x", a.q, a.ldq, rows, k, a.type);
    check_matrix(op, "w", a.p, a.ldp, w_rows, k, a.type);
    check_matrix(op, "out", a.out, a.ldo, rows, n, out_type);
    if (a.resid) check_matrix(op, "resid", a.resid, a.ldr, rows, n, out_type);
    if (a.pre) check_matrix(op, "pre", a.pre, a.ldpre, rows, w_rows, half);
    // The tiles address both halves of Wi by 31-bit offsets from its first row.
    if (a.gated && (n + 256) * k * type_bytes(a.type) >= ((size_t)1 << 31)) refuse(op, "w of 4 GiB or more");
    const Span x = span_of(a.q, a.ldq, rows, k, a.type), w = span_of(a.p, a.ldp, w_rows, k, a.type);
    const Span out = span_of(a.out, a.ldo, rows, n, out_type), pre = span_of(a.pre, a.ldpre, rows, w_rows, half);
    const Span resid = span_of(a.resid, a.ldr, rows, n, out_type);
    check_disjoint(op, "out", out, "x", x);
    check_disjoint(op, "out", out, "w", w);
    check_disjoint(op, "pre", pre, "x", x);
    check_disjoint(op, "pre", pre, "w", w);
    check_disjoint(op, "pre", pre, "out", out);
    check_disjoint(op, "pre", pre, "resid", resid);
    for (const Span& v : {vector_span(a.bias, n), vector_span(a.p_scale, w_rows), vector_span(a.q_scale, rows)}) {
        check_disjoint(op, "out", out, "the bias or a scale", v);
        check_disjoint(op, "pre", pre, "the bias or a scale", v);
    }
    // out may be resid itself: every element is read by the thread that writes it.
    if (a.resid != a.out || a.ldr != a.ldo) check_disjoint(op, "out", out, "resid", resid);
    run(a, plan(op, a, false), nullptr, s);
}

LinearPlan linear_plan(int product, int type, int out_type, size_t rows, size_t n, size_t k) {
    const char* op = "linear_plan";
    if (product < JH_PRODUCT_LINEAR || product > JH_PRODUCT_DW) refuse(op, "unknown product");
    check_sizes(op, type, rows, n, k);
    const bool gradient = product >= JH_PRODUCT_DX;
    const int half = type == JH_E4M3 ? JH_BF16 : type;
    if (gradient && type == JH_E4M3) refuse(op, "gradients are of bf16 or f16 operands");
    if (out_type != half && (out_type != JH_F32 || product == JH_PRODUCT_GATED || product == JH_PRODUCT_DX))
        refuse(op, "no such output type");
    LinearArgs a{};
    a.type = type;
    a.gated = product == JH_PRODUCT_GATED;
    a.out_f32 = out_type == JH_F32;
    a.layout = product == JH_PRODUCT_DX ? COLS_ROWS : product == JH_PRODUCT_DW ? COLS_COLS : ROWS_ROWS;
    a.q_rows = (int)(product == JH_PRODUCT_DW ? n : rows);
    a.p_cols = (int)(gradient ? k : n);
    a.k = (int)(product == JH_PRODUCT_DW ? rows : product == JH_PRODUCT_DX ? n : k);
    const Plan p = plan(op, a, gradient);
    return {{{p.kernel, p.splits, p.whole ? p.whole : a.q_rows}, {p.rest, p.whole ? 1 : 0, p.whole ? a.q_rows - p.whole : 0}}};
}

namespace {

// Workspace of a backward pass: the gradient before the activation, then FP32 parts (of the
// column sums, and after them of the products: the stream runs one after the other).
struct BackwardPlan {
    LinearArgs dx{}, dw{};
    Plan dx_plan{}, dw_plan{};
    long dz_bytes = 0, part_bytes = 0;
    int sum_blocks = 0, rows_per_block = 0;
    size_t bytes() const { return (size_t)(dz_bytes + part_bytes); }
};

BackwardPlan plan_backward(const char* op, int type, size_t rows, size_t n, size_t k, bool keeps_dz, bool sums) {
    BackwardPlan p;
    p.dx.type = p.dw.type = type;
    p.dx.layout = COLS_ROWS;
    p.dx.p_cols = (int)k;
    p.dx.q_rows = (int)rows;
    p.dx.k = (int)n;
    p.dw.layout = COLS_COLS;
    p.dw.p_cols = (int)k;
    p.dw.q_rows = (int)n;
    p.dw.k = (int)rows;
    p.dx_plan = plan(op, p.dx, true);
    p.dw_plan = plan(op, p.dw, true);
    p.dz_bytes = keeps_dz ? round_up((long)rows * n * 2, 256) : 0;
    p.part_bytes = std::max(partial_bytes(p.dx, p.dx_plan), partial_bytes(p.dw, p.dw_plan));
    const long across = (n + 511) / 512, want = std::max(1L, 1024 / across);
    p.rows_per_block = (int)std::max(8L, ((long)rows + want - 1) / want);
    p.sum_blocks = (int)(((long)rows + p.rows_per_block - 1) / p.rows_per_block);
    if (sums) p.part_bytes = std::max(p.part_bytes, round_up((long)p.sum_blocks * n * 4, 256));
    return p;
}

void check_workspace(const char* op, const void* ws, size_t bytes, size_t need) {
    if (need == 0) return;
    if (!ws || ((uintptr_t)ws & 15)) refuse(op, "needs a 16-byte aligned workspace");
    if (bytes < need) refuse(op, "workspace too small");
}

// The two gradient products of a linear layer: dx = dz W and dw = dzᵀ x.
void run_products(const BackwardPlan& p, const void* dz, long lddz, const LinearGradArgs& a, float* partial,
                  hipStream_t s) {
    if (a.dx && p.dx.q_rows) {
        LinearArgs d = p.dx;
        d.p = a.w;
        d.ldp = p.dx.p_cols;
        d.q = dz;
        d.ldq = lddz;
        d.out = a.dx;
        d.ldo = a.lddx;
        run(d, p.dx_plan, partial, s);
    }
    if (a.dw) {
        LinearArgs d = p.dw;
        d.p = a.x;
        d.ldp = a.ldx;
        d.q = dz;
        d.ldq = lddz;
        d.out = a.dw;
        d.ldo = p.dw.p_cols;
        d.out_f32 = a.grad_f32;
        run(d, p.dw_plan, partial, s);
    }
}

}  // namespace

size_t linear_backward_workspace(size_t rows, size_t n, size_t k, int act, bool gated) {
    const char* op = gated ? "gated_ffn_backward" : "linear_backward";
    check_sizes(op, JH_BF16, rows, n, k);
    if (gated && n % 16) refuse(op, "output features must be a multiple of 8");
    check_act(op, act);
    return plan_backward(op, JH_BF16, rows, n, k, gated || act != JH_ACT_NONE, !gated).bytes();
}

void linear_backward(const LinearGradArgs& args, size_t rows, size_t n, size_t k, hipStream_t s) {
    LinearGradArgs a = args;
    const char* op = a.gated ? "gated_ffn_backward" : "linear_backward";
    if (a.type == JH_E4M3) refuse(op, "gradients are of bf16 or f16 operands");
    check_sizes(op, a.type, rows, n, k);
    check_act(op, a.act);
    const size_t inter = n / 2, dy_cols = a.gated ? inter : n;
    if (a.gated && n % 16) refuse(op, "output features must be a multiple of 8");
    const bool keeps_dz = a.gated || a.act != JH_ACT_NONE;
    const int grad_type = a.grad_f32 ? JH_F32 : a.type;
    if (!a.dx && !a.dw && !a.dbias) refuse(op, "no gradient asked for");
    a.lddy = row_stride(a.lddy, rows, dy_cols);
    a.ldpre = row_stride(a.ldpre, rows, n);
    a.ldx = row_stride(a.ldx, rows, k);
    a.lddx = row_stride(a.lddx, rows, k);
    const BackwardPlan p = plan_backward(op, a.type, rows, n, k, keeps_dz, a.dbias != nullptr);
    check_workspace(op, a.workspace, a.workspace_bytes, p.bytes());
    const Span ws = span_of(a.workspace, p.bytes(), p.bytes() ? 1 : 0, p.bytes(), JH_E4M3);
    if (rows) check_matrix(op, a.gated ? "dh" : "dy", a.dy, a.lddy, rows, dy_cols, a.type);
    if (rows && keeps_dz) check_matrix(op, a.gated ? "gu" : "pre", a.pre, a.ldpre, rows, n, a.type);
    if (a.dx && rows) {
        check_matrix(op, "w", a.w, k, n, k, a.type);
        check_matrix(op, "dx", a.dx, a.lddx, rows, k, a.type);
    }
    if (a.dw) {
        if (rows) check_matrix(op, "x", a.x, a.ldx, rows, k, a.type);
        check_matrix(op, "dw", a.dw, k, n, k, grad_type);
    }
    const Span in[4] = {span_of(a.dy, a.lddy, rows, dy_cols, a.type),
                        span_of(keeps_dz ? a.pre : nullptr, a.ldpre, rows, n, a.type),
                        span_of(a.dw ? a.x : nullptr, a.ldx, rows, k, a.type),
                        span_of(a.dx ? a.w : nullptr, k, n, k, a.type)};
    const Span out[4] = {span_of(a.dx, a.lddx, rows, k, a.type), span_of(a.dw, k, n, k, grad_type),
                         span_of(a.dbias, n, 1, n, JH_F32), ws};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 4; ++i) check_disjoint(op, "an output or the workspace", out[o], "an input", in[i]);
        for (int i = 0; i < o; ++i) check_disjoint(op, "an output", out[o], "another", out[i]);
    }

    uint8_t* const base = (uint8_t*)a.workspace;
    float* const partial = (float*)(base + p.dz_bytes);
    const void* dz = a.dy;
    long lddz = a.lddy;
    if (keeps_dz) {
        dz = base;
        lddz = (long)n;
    }
    if (a.gated && rows) {
        const GatedGradArgs g{a.dy, a.lddy, a.pre, a.ldpre, base, (int)rows, (int)inter, a.act};
        const dim3 grid(blocks_of((long)rows * (inter / 8), op));
        if (a.type == JH_BF16) JH_LAUNCH(gated_grad_kernel<Bf16>, grid, dim3(THREADS), 0, s, g);
        else JH_LAUNCH(gated_grad_kernel<F16>, grid, dim3(THREADS), 0, s, g);
        HIP_CHECK(hipGetLastError());
    } else if (!a.gated && (keeps_dz || a.dbias)) {
        if (rows) {
            const ActGradArgs g{a.dy, a.lddy, keeps_dz ? a.pre : nullptr, a.ldpre, base, a.dbias ? partial : nullptr,
                                (int)rows, (int)n, p.rows_per_block, a.act};
            const dim3 grid((unsigned)((n + 511) / 512), (unsigned)p.sum_blocks);
            if (a.type == JH_BF16) JH_LAUNCH(act_grad_kernel<Bf16>, grid, dim3(THREADS), 0, s, g);
            else JH_LAUNCH(act_grad_kernel<F16>, grid, dim3(THREADS), 0, s, g);
            HIP_CHECK(hipGetLastError());
        }
        if (a.dbias) launch_column_sum(partial, p.sum_blocks, (int)n, a.dbias, s);
    }
    run_products(p, dz, lddz, a, partial, s);
}
