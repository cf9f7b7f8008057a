// Rows in 8-bit integers: q = rint(v * (127 / m)) with m the row's largest |v|, and the row's scale in 32 bits, scale * q ~ v.
// What the 8-bit product reads (int8_product.cu). The values v come from
//   rows        v = x
//   norm        x <- x + add (optional), v = x * weight; the scale also takes the norm's factor 1 / sqrt(mean(x^2) + eps)
//   activation  v = act(g) * u of a row [g; u], rounded to bfloat16 as the bfloat16 path has it
//
// The norm's factor is the same for the whole row, so the integers do not depend on it: the sum of squares and the largest value
// are found in the same pass and meet in one exchange between the warps, and every thread keeps its values in registers. A pass
// reads the row once and writes a quarter of it (all of it again where the sum goes back): memory bound for many rows, one exchange
// and the launch for few. The integers take three operations that IEEE arithmetic fixes (a product, a quotient per row, a product), so
// they do not depend on how a row is cut over threads.
//
// What is not finite: the largest |v| is kept as the bits of its absolute value, an integer that orders infinities and NaN above
// every number, so that one of them anywhere in a row shows: such a row gets the scale NaN and zeros, and every product with it is
// NaN. A norm whose squares or products with the weights leave the range of 32 bits is taken again: the squares from values 2^-80 times as large, or
// 2^80 times where they vanish beside an eps that is as small, and the products with the weights likewise, each by a factor of its own (values near 1 with weights
// near 2^127 have squares as they should be).
// Rows whose largest |v| (as it was taken last) is below 2^-100 count as zero (scale 0): 127 / m would leave that range at the other end.
#include "common.cuh"

namespace gi {
namespace {

enum RowsKind : int { kRowsPlain = 0, kRowsNorm = 1, kRowsGated = 2 };

struct RowsParams {
    const void* x;          // rows of D values (gated: 2 D), ldx values apart; the norm's are 32-bit and written where add is
    const void* add;        // norm: [T, D] or null
    const float* weight;    // norm: [D]; gated: the bias [2 D] or null
    int8_t* q;              // [T, width]
    float* scales;          // [T]
    long long ldx;
    int T, D, width;        // width: D or more, a multiple of 16; zeros behind D
    int act;
    float limit, eps;
    int w_constant;         // norm: no kernel that may still be running writes weight: it may be read before the wait
};

constexpr unsigned kInfBits = 0x7f800000u, kLeastBits = 0x0d800000u, kSmallBits = 0x35800000u;      // 2^-100, 2^-20
constexpr float kDown = 8.271806125530277e-25f, kUp = 1.2089258196146292e24f;      // 2^-80, 2^80
constexpr float kLeastSquares = 7.888609052210118e-31f, kLeastEps = 7.52316384526264e-37f;      // 2^-100, 2^-120

// Four values of a row to a thread. VEC: neighbours, at 4 i, one access of 16 (8) bytes; rows of any width and alignment: at i, i + G, i + 2 G,
// i + 3 G, so that the lanes of a warp stay side by side (2048 rows of 2050: 43 us with four neighbours one by one, 15.7 with these; of 2048: 9).
template <bool VEC, int G>
__device__ __forceinline__ int column(int i, int j) { return VEC ? 4 * i + j : (i / G) * 4 * G + i % G + j * G; }

template <bool VEC, int G>
__device__ __forceinline__ float4 load4(const float* p, int i, int D) {
    if constexpr (VEC) {
        return 4 * i < D ? *reinterpret_cast<const float4*>(p + 4 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = column<VEC, G>(i, j) < D ? p[column<VEC, G>(i, j)] : 0.f;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
}
template <bool VEC, int G>
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p, int i, int D) {
    if constexpr (VEC) {
        if (4 * i >= D) return make_float4(0.f, 0.f, 0.f, 0.f);
        const uint2 raw = *reinterpret_cast<const uint2*>(p + 4 * i);
        return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                           __uint_as_float(raw.y & 0xffff0000u));
    } else {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = column<VEC, G>(i, j) < D ? to_float(p[column<VEC, G>(i, j)]) : 0.f;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
}
template <bool VEC, int G>
__device__ __forceinline__ void store4(float* p, int i, int D, const float4 v) {
    if constexpr (VEC) {
        if (4 * i < D) *reinterpret_cast<float4*>(p + 4 * i) = v;
    } else {
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (column<VEC, G>(i, j) < D) p[column<VEC, G>(i, j)] = e[j];
    }
}

struct NoAdd {};        // a norm without an addition

// What a norm's values are multiplied by ahead of their squares and ahead of the weights.
struct Factors { float squares = 1.f, values = 1.f; };

__device__ __forceinline__ float4 plus(const float4 a, const float4 b) {
    return make_float4(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y), __fadd_rn(a.z, b.z), __fadd_rn(a.w, b.w));
}

// N groups of four values of a row, i0, i0 + G, ..: v of each, and what the squares add to ss. All loads stand before the first
// store of a row that is written back (nothing tells the compiler that they do not overlap). `first`: the norm's addition is done. Only the first
// `live` groups have columns for any thread: activations of the others are skipped, by all threads at once (14,336 values in 512 x 8 groups of four: an
// eighth). Their loads are not: they are masked anyway, and a branch between loads keeps them from being under way together.
template <int KIND, typename TX, typename TA, bool VEC, int G, int N>
__device__ __forceinline__ void values(const RowsParams& p, long long row, int i0, int live, const float4* w, const Factors factor, bool first, float& ss, float4* v) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = load4<VEC, G>(x, i0 + k * G, p.D);
    if constexpr (KIND == kRowsGated) {
        float4 u[N];
#pragma unroll
        for (int k = 0; k < N; ++k) u[k] = load4<VEC, G>(x + p.D, i0 + k * G, p.D);
        if (p.weight != nullptr) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = plus(v[k], load4<VEC, G>(p.weight, i0 + k * G, p.D));
                u[k] = plus(u[k], load4<VEC, G>(p.weight + p.D, i0 + k * G, p.D));
            }
        }
        with_activation(p.act, [&](auto act) {
            auto h = [&](float g, float up) { return gated_value_bf16<decltype(act)::value>(g, up, p.limit); };
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (k >= live) continue;
                const __nv_bfloat162 lo = __floats2bfloat162_rn(h(v[k].x, u[k].x), h(v[k].y, u[k].y));
                const __nv_bfloat162 hi = __floats2bfloat162_rn(h(v[k].z, u[k].z), h(v[k].w, u[k].w));
                const uint32_t a = *reinterpret_cast<const uint32_t*>(&lo), b = *reinterpret_cast<const uint32_t*>(&hi);
                v[k] = make_float4(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
            }
        });
    } else if constexpr (KIND == kRowsNorm) {
        if constexpr (!std::is_same<TA, NoAdd>::value) {
            if (first) {
                float4 a[N];
#pragma unroll
                for (int k = 0; k < N; ++k) a[k] = load4<VEC, G>(static_cast<const TA*>(p.add) + row * p.D, i0 + k * G, p.D);
#pragma unroll
                for (int k = 0; k < N; ++k) v[k] = plus(v[k], a[k]);
#pragma unroll
                for (int k = 0; k < N; ++k) store4<VEC, G>(static_cast<float*>(const_cast<void*>(p.x)) + row * p.ldx, i0 + k * G, p.D, v[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            auto times = [&](float f) { return make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f); };
            const float4 e = times(factor.squares), x = times(factor.values);
            ss = fmaf(e.x, e.x, ss); ss = fmaf(e.y, e.y, ss); ss = fmaf(e.z, e.z, ss); ss = fmaf(e.w, e.w, ss);
            v[k] = make_float4(__fmul_rn(x.x, w[k].x), __fmul_rn(x.y, w[k].y), __fmul_rn(x.z, w[k].z), __fmul_rn(x.w, w[k].w));
        }
    }
}

// rint(v * inv) of |v * inv| <= 127.5 in the low byte: the sum with 1.5 * 2^23 is rounded to a whole number, to the even one of two (an addition, where
// the conversion to an integer takes the unit that exponentials take, a quarter as wide).
__device__ __forceinline__ uint32_t int_of(float v, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); }

template <bool VEC, int G>
__device__ __forceinline__ void put4(int8_t* q, int i, int width, const float4 v, float inv, bool none) {
    const uint32_t a = int_of(v.x, inv), b = int_of(v.y, inv), c = int_of(v.z, inv), d = int_of(v.w, inv);
    if constexpr (VEC) {
        if (4 * i < width) reinterpret_cast<uint32_t*>(q)[i] = none ? 0u : __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    } else {
        const uint32_t e[4] = {a, b, c, d};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (column<VEC, G>(i, j) < width) q[column<VEC, G>(i, j)] = none ? 0 : static_cast<int8_t>(e[j] & 0xffu);
    }
}

__device__ __forceinline__ unsigned top_bits(const float4 v, unsigned m) {
    m = max(m, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
    return max(m, max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
}

// The factors that a norm has to be taken again with; false: it is right as it is. (Products below 2^-20 of values that are small enough for kUp: none above
// 2^60 then.)
__device__ __forceinline__ bool other_factors(unsigned m, float ss, float eps, Factors& f) {
    if (!(ss < __uint_as_float(kInfBits))) f.squares = kDown;
    else if (ss < kLeastSquares && eps < kLeastEps) f.squares = kUp;
    if (m >= kInfBits) f.values = kDown;
    else if (f.squares == kUp && m < kSmallBits) f.values = kUp;
    return f.squares != 1.f || f.values != 1.f;
}

// The row's largest |v| and sum of squares over the G threads that share it.
template <int G, int KIND>
__device__ __forceinline__ void meet(unsigned& m, float& ss, unsigned* part_m, float* part_s) {
    m = __reduce_max_sync(0xffffffffu, m);
    if (KIND == kRowsNorm) ss = warp_sum(ss);
    if (G > 32) {
        constexpr int kWarps = G / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) { part_m[warp] = m; part_s[warp] = ss; }
        __syncthreads();
        m = lane < kWarps ? part_m[lane] : 0u;
        m = __reduce_max_sync(0xffffffffu, m);
        if (KIND == kRowsNorm) ss = warp_sum(lane < kWarps ? part_s[lane] : 0.f);
    }
}

// 127 / m and the scale of a row; a row that is not finite: 0 and NaN.
template <int KIND>
__device__ __forceinline__ float2 row_factors(unsigned m_bits, float ss, const RowsParams& p, const Factors factor) {
    if (m_bits >= kInfBits || (KIND == kRowsNorm && !(ss < __uint_as_float(kInfBits)))) return make_float2(0.f, __uint_as_float(0x7fc00000u));
    if (m_bits < kLeastBits) return make_float2(0.f, 0.f);
    const float m = __uint_as_float(m_bits);
    float scale = __fdiv_rn(m, 127.f);
    // (squares of values f times as large: their mean and eps are both f^2 times as large, the root f times; powers of two are exact)
    if (KIND == kRowsNorm) {
        const float f = factor.squares, root = sqrtf(__fdiv_rn(ss, static_cast<float>(p.D)) + p.eps * f * f);
        scale = __fdiv_rn(scale, root);
        if (f != factor.values) scale *= f > factor.values ? kUp : kDown;      // f / values: 2^80 or 2^-80, as they never lie further apart
    }
    return make_float2(__fdiv_rn(127.f, m), scale);
}

// G threads to a row, V groups of four values each in registers, read in batches: 64 registers, so that an SM holds 1,024 threads of it (of two rows at least,
// up to 16,384 values). 8,192 rows of 4,096 with a 32-bit addition: 64 us, 6.8 TB/s (the measured copy rate is 6.55; some of it stays in L2); 8,192 of 16,384
// from 16 bits: 78 us, 5.1 TB/s; 4,096 activated rows of 14,336: from 32 bits 90 us, 5.9 TB/s, from 16 bits 67 us, 4.4 TB/s (neither memory, at half its rate, nor
// the issue of instructions, 23 a value at 2.3 of 4 a cycle, is full: a row's loads, arithmetic and stores follow each other, and two rows are all that an SM holds).
// One row of 2,048: 1.8 us in a stream of launches.
template <int KIND, typename TX, typename TA, int G, int V, bool VEC>
__global__ void __launch_bounds__(G < 128 ? 128 : G, G <= 512 ? 1024 / (G < 128 ? 128 : G) : 1)
rows_int8_kernel(const RowsParams p) {
    constexpr int kRows = G < 128 ? 128 / G : 1;
    constexpr int kBatch = V <= 4 ? V : sizeof(TX) == 2 ? 4 : 2;      // (16-bit values wait in half the registers)
    constexpr bool kHeld = V <= 4;       // registers hold all of a thread's weights of a norm: constant ones are read before the wait for the kernel ahead
    __shared__ unsigned part_m[2][32];
    __shared__ float part_s[2][32];
    const int t = threadIdx.x % G;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G;
    const int live = (p.width + 4 * G - 1) / (4 * G);
    if (threadIdx.x == 0) timeline_record(kTlInt8Rows, 0);
    pdl_launch_dependents();
    float4 w[kBatch];
    auto weights = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) w[k] = KIND == kRowsNorm ? load4<VEC, G>(p.weight, t + (k0 + k) * G, p.D) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    if (kHeld && p.w_constant) weights(0);
    pdl_wait();
    if (threadIdx.x == 0) timeline_record(kTlInt8Rows, 1);
    if (row >= p.T) return;       // (whole warps: rows of several to a block have a warp each)
    if (kHeld && !p.w_constant) weights(0);
    float4 v[V];
    unsigned m = 0;
    float ss = 0.f;
    Factors factor;
#pragma unroll
    for (int k = 0; k < V; k += kBatch) {
        if (!kHeld) weights(k);
        values<KIND, TX, TA, VEC, G, kBatch>(p, row, t + k * G, live - k, w, factor, true, ss, v + k);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) m = top_bits(v[k], m);
    meet<G, KIND>(m, ss, part_m[0], part_s[0]);
    if (KIND == kRowsNorm && other_factors(m, ss, p.eps, factor)) {
        m = 0;
        ss = 0.f;
#pragma unroll
        for (int k = 0; k < V; k += kBatch) {
            if (!kHeld) weights(k);
            values<KIND, TX, TA, VEC, G, kBatch>(p, row, t + k * G, live - k, w, factor, false, ss, v + k);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) m = top_bits(v[k], m);
        meet<G, KIND>(m, ss, part_m[1], part_s[1]);
    }
    const float2 f = row_factors<KIND>(m, ss, p, factor);
    const bool none = f.x == 0.f;        // (0 * infinity would not be 0)
#pragma unroll
    for (int k = 0; k < V; ++k) put4<VEC, G>(p.q + row * p.width, t + k * G, p.width, v[k], f.x, none);
    if (t == 0) p.scales[row] = f.y;
    if (threadIdx.x == 0) timeline_record(kTlInt8Rows, 6);
}

// Rows wider than a block's registers: the same twice over memory.
template <int KIND, typename TX, typename TA>
__global__ void __launch_bounds__(1024)
wide_rows_int8_kernel(const RowsParams p) {
    __shared__ unsigned part_m[2][32];
    __shared__ float part_s[2][32];
    const long long row = blockIdx.x;
    pdl_prologue();
    unsigned m = 0;
    float ss = 0.f;
    Factors factor;
    float4 v[1], w[1];
    auto pass = [&](int i, bool first, float& squares) {
        w[0] = KIND == kRowsNorm ? load4<false, 1024>(p.weight, i, p.D) : make_float4(0.f, 0.f, 0.f, 0.f);
        values<KIND, TX, TA, false, 1024, 1>(p, row, i, 1, w, factor, first, squares, v);
    };
    const int groups = (p.width + 4095) / 4096 * 1024;
    for (int i = threadIdx.x; i < groups; i += 1024) { pass(i, true, ss); m = top_bits(v[0], m); }
    meet<1024, KIND>(m, ss, part_m[0], part_s[0]);
    if (KIND == kRowsNorm && other_factors(m, ss, p.eps, factor)) {
        m = 0;
        ss = 0.f;
        for (int i = threadIdx.x; i < groups; i += 1024) { pass(i, false, ss); m = top_bits(v[0], m); }
        meet<1024, KIND>(m, ss, part_m[1], part_s[1]);
    }
    const float2 f = row_factors<KIND>(m, ss, p, factor);
    const bool none = f.x == 0.f;
    float unused = 0.f;
    for (int i = threadIdx.x; i < groups; i += 1024) {
        pass(i, false, unused);
        put4<false, 1024>(p.q + row * p.width, i, p.width, v[0], f.x, none);
    }
    if (threadIdx.x == 0) p.scales[row] = f.y;
}

template <int KIND, typename TX, typename TA, bool VEC>
void launch_rows(const RowsParams& p, cudaStream_t st) {
    auto go = [&](auto* kernel, int threads, int rows) {
        launch_kernel(kernel, dim3(static_cast<unsigned>((static_cast<long long>(p.T) + rows - 1) / rows)), dim3(threads), 0, st, p);
    };
    if (p.width <= 512) go(rows_int8_kernel<KIND, TX, TA, 32, 4, VEC>, 128, 4);
    else if (p.width <= 2048) go(rows_int8_kernel<KIND, TX, TA, 128, 4, VEC>, 128, 1);
    else if (p.width <= 4096) go(rows_int8_kernel<KIND, TX, TA, 256, 4, VEC>, 256, 1);
    else if (p.width <= 8192) go(rows_int8_kernel<KIND, TX, TA, 512, 4, VEC>, 512, 1);
    else if (p.width <= 16384) {
        if (VEC) go(rows_int8_kernel<KIND, TX, TA, 512, 8, true>, 512, 1);      // two rows to an SM: one is read while the other is written
        else go(rows_int8_kernel<KIND, TX, TA, 1024, 4, false>, 1024, 1);       // (512 threads lack the registers)
    }
    else if (p.width <= 32768) go(rows_int8_kernel<KIND, TX, TA, 1024, 8, VEC>, 1024, 1);
    else go(wide_rows_int8_kernel<KIND, TX, TA>, 1024, 1);
}

template <int KIND, typename TX, typename TA>
int run_rows(const RowsParams& p, bool vec, cudaStream_t st) {
    if (vec) launch_rows<KIND, TX, TA, true>(p, st);
    else launch_rows<KIND, TX, TA, false>(p, st);
    return check_launch("rows_int8");
}

// 16 bytes of 32-bit values, 8 of bfloat16: whole groups of four
bool aligned4(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == kF32 ? 16 : 8) == 0; }

int rows_int8_impl(int kind, const void* x, int x_dtype, long long ldx, const void* add, int add_dtype, const float* weight, float eps, int act,
                   float limit, void* q, int width, float* scales, int T, int D, int w_constant, void* stream) {
    if (T == 0) return 0;
    GI_REQUIRE(T > 0 && D > 0, "rows_int8: sizes must be positive (rows=%d, D=%d)", T, D);
    GI_REQUIRE(D <= (1 << 30), "rows_int8: rows of %d values (at most 2^30)", D);
    GI_REQUIRE(width % 16 == 0 && width >= D && width - D < 16, "rows_int8: the output's width %d must be the multiple of 16 that follows %d", width, D);
    GI_REQUIRE(x_dtype == kF32 || x_dtype == kBF16, "rows_int8: unsupported dtype code %d", x_dtype);
    GI_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0, "rows_int8: the output must be 16-byte aligned");
    GI_REQUIRE(act >= 0 && act < kActCount, "rows_int8: unknown activation %d", act);
    GI_REQUIRE(!(act == kActCappedSwish && limit < 0.f), "rows_int8: a bound of %g (not below zero: zeros behind a row have to stay zeros)", limit);
    GI_REQUIRE(ldx >= (kind == kRowsGated ? 2ll : 1ll) * D || T == 1, "rows_int8: rows of x overlap");
    const RowsParams p{x, add, weight, static_cast<int8_t*>(q), scales, ldx, T, D, width, act, limit, eps, w_constant};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    bool vec = D % 4 == 0 && (ldx % 4 == 0 || T == 1) && aligned4(x, x_dtype) && (weight == nullptr || aligned4(weight, kF32));
    if (kind == kRowsNorm) {
        GI_REQUIRE(x_dtype == kF32 && weight != nullptr, "rows_int8: a norm takes 32-bit rows and weights");
        if (add == nullptr) return run_rows<kRowsNorm, float, NoAdd>(p, vec, st);
        GI_REQUIRE(add_dtype == kF32 || add_dtype == kBF16, "rows_int8: unsupported dtype code %d", add_dtype);
        vec = vec && aligned4(add, add_dtype);
        return add_dtype == kF32 ? run_rows<kRowsNorm, float, float>(p, vec, st) : run_rows<kRowsNorm, float, __nv_bfloat16>(p, vec, st);
    }
    if (kind == kRowsGated)
        return x_dtype == kF32 ? run_rows<kRowsGated, float, NoAdd>(p, vec, st) : run_rows<kRowsGated, __nv_bfloat16, NoAdd>(p, vec, st);
    GI_REQUIRE(kind == kRowsPlain, "rows_int8: unknown kind %d", kind);
    return x_dtype == kF32 ? run_rows<kRowsPlain, float, NoAdd>(p, vec, st) : run_rows<kRowsPlain, __nv_bfloat16, NoAdd>(p, vec, st);
}

}  // namespace
}  // namespace gi
GI_TIMELINE_SETTER(gi_timeline_set_int8_rows)

// q [T, width] and scales [T] of T rows: kind 0 of x [T, D], 1 of the norm of x (32-bit; x += add [T, D] first where add is given), 2 of
// act(g) * u with x [T, 2 D] = [g; u] and `weight` its bias (may be null). Rows of x lie ldx values apart. w_constant: no launch before this one that may
// still be running writes the norm's `weight`, so that it may be read before the wait for them.
extern "C" int gi_rows_int8(int kind, const void* x, int x_dtype, long long ldx, const void* add, int add_dtype, const float* weight, float eps,
                            int act, float limit, void* q, int width, float* scales, int T, int D, int w_constant, void* stream) {
    return gi::dispatch(gi::rows_int8_impl, kind, x, x_dtype, ldx, add, add_dtype, weight, eps, act, limit, q, width, scales, T, D, w_constant, stream);
}
