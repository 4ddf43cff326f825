// Activations that keep their input in 8 bits, and their backward pass from what was kept (formats: lowbit_formats.h).
#include "lowbit_internal.h"

namespace cntkq {
namespace lowbit {

namespace {

constexpr uint32_t kThreads = 256;

// e^x for values that come from or go to the element type. The device's exponential takes a power of two, and the product with log2 e is rounded by up to half a
// place of itself: an error of |x| 2^-25 of the result and more, 4e-6 for x = 80. In single precision what the rounded power leaves of x is multiplied on,
// with ln 2 in two parts, and 2e-7 are left anywhere; half precision and bfloat16 round their results by far more.
template <int DT>
__device__ __forceinline__ float exponential(float x)
{
    if constexpr (DT != kF32)
        return __expf(x);
    const float p = x * 1.44269504f, y = __builtin_amdgcn_exp2f(p);
    const float rest = __builtin_fmaf(p, 1.90465430e-9f, __builtin_fmaf(p, -0.693147182f, x)); // x - p ln 2
    return __builtin_fabsf(p) < 128.0f ? __builtin_fmaf(y, rest, y) : y; // (0 or infinite beyond)
}

// The function, in 32 bits.
template <int KIND, int DT>
__device__ __forceinline__ float activate(float x)
{
    if constexpr (KIND == kSigmoid)
        return 1.0f / (1.0f + exponential<DT>(-x));
    else if constexpr (KIND == kTanh)
        return tanhf(x);
    else if constexpr (KIND == kRelu)
        return x < 0.0f ? 0.0f : x; // (a NaN stays one)
    else if constexpr (KIND == kGelu)
        return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    else if constexpr (KIND == kSilu)
        return x / (1.0f + exponential<DT>(-x));
    else
        return x;
}

// The function and its derivative.
template <int KIND, int DT>
__device__ __forceinline__ void activate_slope(float x, float& f, float& d)
{
    if constexpr (KIND == kSigmoid)
    {
        f = 1.0f / (1.0f + exponential<DT>(-x));
        d = f * (1.0f - f);
    }
    else if constexpr (KIND == kTanh)
    {
        f = tanhf(x);
        d = 1.0f - f * f;
    }
    else if constexpr (KIND == kRelu)
    {
        f = x < 0.0f ? 0.0f : x;
        d = x > 0.0f ? 1.0f : (x <= 0.0f ? 0.0f : x);
    }
    else if constexpr (KIND == kGelu)
    {
        const float phi = 0.5f * (1.0f + erff(x * 0.70710678118654752f));
        f = x * phi;
        d = phi + x * exponential<DT>(-0.5f * x * x) * 0.39894228040143268f;
    }
    else if constexpr (KIND == kSilu)
    {
        const float s = 1.0f / (1.0f + exponential<DT>(-x));
        f = x * s;
        d = s * (1.0f + x * (1.0f - s));
    }
    else
    {
        f = x;
        d = 1.0f;
    }
}

// Rows are dealt to groups of 2^lanes_log threads, eight values a thread (four neighbouring lanes have a block).
struct RowGrid
{
    uint32_t rows, cols, pitch, lanes_log, chunks;
};
RowGrid row_grid(size_t rows, size_t cols)
{
    RowGrid g;
    g.rows = (uint32_t) rows;
    g.cols = (uint32_t) cols;
    g.pitch = (uint32_t) save8_pitch(cols);
    g.lanes_log = 2;
    while (g.lanes_log < 8 && (8u << g.lanes_log) < g.pitch)
        ++g.lanes_log;
    g.chunks = (uint32_t) ceil_div(g.pitch, (size_t) 8 << g.lanes_log);
    return g;
}
uint32_t row_blocks(const RowGrid& g)
{
    return (uint32_t) ceil_div(g.rows, kThreads >> g.lanes_log) * g.chunks;
}
struct Place
{
    uint32_t row, col;
    int valid;
    bool inside; // of the padded matrix
};
__device__ __forceinline__ Place place(const RowGrid& g)
{
    Place p;
    p.row = (blockIdx.x / g.chunks) * (kThreads >> g.lanes_log) + (threadIdx.x >> g.lanes_log);
    p.col = (((blockIdx.x % g.chunks) << g.lanes_log) + (threadIdx.x & ((1u << g.lanes_log) - 1))) * 8;
    p.inside = p.row < g.rows && p.col < g.pitch;
    p.valid = p.inside && p.col < g.cols ? (int) min(g.cols - p.col, 8u) : 0;
    return p;
}

template <int DT>
__device__ __forceinline__ const typename Type<DT>::T* row_of(const RowGrid& g, const Place& p, const void* base, int64_t stride)
{
    return static_cast<const typename Type<DT>::T*>(base) + (int64_t) min(p.row, g.rows - 1) * stride;
}
__device__ __forceinline__ void keep(const RowGrid& g, const Place& p, const float (&v)[8], void* saved)
{
    const uint32_t s = save8_scale(quad_max(top8(v)));
    if (!p.inside)
        return;
    int8_t* codes = static_cast<int8_t*>(saved);
    *reinterpret_cast<u32x2*>(codes + (size_t) p.row * g.pitch + p.col) = save8_encode8(v, s);
    if (p.col % kBlock == 0)
        reinterpret_cast<uint8_t*>(codes + (size_t) g.rows * g.pitch)[(size_t) p.row * (g.pitch / kBlock) + p.col / kBlock] = (uint8_t) s;
}
struct Kept
{
    u32x2 codes;
    uint32_t scale;
};
__device__ __forceinline__ void fetch(const RowGrid& g, const Place& p, const void* saved, Kept& k)
{
    const int8_t* codes = static_cast<const int8_t*>(saved);
    k.scale = reinterpret_cast<const uint8_t*>(codes + (size_t) g.rows * g.pitch)[(size_t) p.row * (g.pitch / kBlock) + p.col / kBlock];
    k.codes = *reinterpret_cast<const u32x2*>(codes + (size_t) p.row * g.pitch + p.col);
}

// y = f(x), or f(gate) x; x (and the gate) kept in 8 bits. Bound by memory: each value read once, written once, 33/32 bytes kept.
// Gated, 8192 x 4096 in bfloat16: 271 MB in 52 us, 5.2 TB/s, a large copy's rate; 1024 x 2048 in single precision 6.1 us.
template <int KIND, int DT, bool GATED, bool WHOLE>
__global__ __launch_bounds__(kThreads) void activation_forward_kernel(ActivationForward a, RowGrid g)
{
    const Place p = place(g);
    const bool there = p.row < g.rows;
    Raw8<DT, WHOLE> raw_x, raw_gate;
    fetch8<DT, WHOLE>(row_of<DT>(g, p, a.x, a.x_stride), p.col, g.cols, raw_x);
    if constexpr (GATED)
        fetch8<DT, WHOLE>(row_of<DT>(g, p, a.gate, a.gate_stride), p.col, g.cols, raw_gate);
    float x[8], gate[8];
    up8<DT, WHOLE>(raw_x, p.col, g.cols, there, x);
    if constexpr (GATED)
        up8<DT, WHOLE>(raw_gate, p.col, g.cols, there, gate);
    keep(g, p, x, a.saved_x);
    if constexpr (GATED)
        keep(g, p, gate, a.saved_gate);
    if constexpr (KIND != kNone)
    {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = GATED ? activate<KIND, DT>(gate[i]) * x[i] : activate<KIND, DT>(x[i]);
        if (p.valid > 0)
            store8<DT>(a.y, (size_t) ((int64_t) p.row * a.y_stride) + p.col, p.valid, y);
    }
}

// dx = dy f'(x8); gated dx = dy f(g8), dgate = dy x8 f'(g8). Bound by memory: 270 MB in 48 us,
// and 6.0 us, for the matrices above.
template <int KIND, int DT, bool GATED, bool WHOLE>
__global__ __launch_bounds__(kThreads) void activation_backward_kernel(ActivationBackward a, RowGrid g)
{
    const Place p = place(g);
    if (p.valid == 0)
        return;
    float dy[8], x[8], dx[8];
    Raw8<DT, WHOLE> raw;
    Kept kept_x, kept_gate;
    fetch8<DT, WHOLE>(row_of<DT>(g, p, a.dy, a.dy_stride), p.col, g.cols, raw);
    fetch(g, p, a.saved_x, kept_x);
    if constexpr (GATED)
        fetch(g, p, a.saved_gate, kept_gate);
    up8<DT, WHOLE>(raw, p.col, g.cols, true, dy);
    save8_decode8(kept_x.codes, kept_x.scale, x);
    if constexpr (GATED)
    {
        float gate[8], dgate[8];
        save8_decode8(kept_gate.codes, kept_gate.scale, gate);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            float f, d;
            activate_slope<KIND, DT>(gate[i], f, d);
            dx[i] = dy[i] * f;
            dgate[i] = dy[i] * x[i] * d;
        }
        store8<DT>(a.dgate, (size_t) ((int64_t) p.row * a.dgate_stride) + p.col, p.valid, dgate);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            float f, d;
            activate_slope<KIND, DT>(x[i], f, d);
            dx[i] = dy[i] * d;
        }
    }
    store8<DT>(a.dx, (size_t) ((int64_t) p.row * a.dx_stride) + p.col, p.valid, dx);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void load8_kernel(const void* saved, void* out, int64_t stride, RowGrid g)
{
    const Place p = place(g);
    if (p.valid == 0)
        return;
    Kept kept;
    fetch(g, p, saved, kept);
    float v[8];
    save8_decode8(kept.codes, kept.scale, v);
    store8<DT>(out, (size_t) ((int64_t) p.row * stride) + p.col, p.valid, v);
}

template <int KIND, int DT, bool GATED>
hipError_t forward(hipStream_t s, const ActivationForward& a)
{
    const RowGrid g = row_grid(a.rows, a.cols);
    if (a.cols % 8 == 0)
        activation_forward_kernel<KIND, DT, GATED, true><<<row_blocks(g), kThreads, 0, s>>>(a, g);
    else
        activation_forward_kernel<KIND, DT, GATED, false><<<row_blocks(g), kThreads, 0, s>>>(a, g);
    return hipGetLastError();
}
template <int KIND, int DT>
hipError_t forward(hipStream_t s, const ActivationForward& a)
{
    return a.gate != nullptr ? forward<KIND, DT, true>(s, a) : forward<KIND, DT, false>(s, a);
}
template <int KIND, int DT, bool GATED>
hipError_t backward(hipStream_t s, const ActivationBackward& a)
{
    const RowGrid g = row_grid(a.rows, a.cols);
    if (a.cols % 8 == 0)
        activation_backward_kernel<KIND, DT, GATED, true><<<row_blocks(g), kThreads, 0, s>>>(a, g);
    else
        activation_backward_kernel<KIND, DT, GATED, false><<<row_blocks(g), kThreads, 0, s>>>(a, g);
    return hipGetLastError();
}
template <int KIND, int DT>
hipError_t backward(hipStream_t s, const ActivationBackward& a)
{
    return a.saved_gate != nullptr ? backward<KIND, DT, true>(s, a) : backward<KIND, DT, false>(s, a);
}

template <int DT>
struct Forward
{
    static hipError_t run(hipStream_t s, int kind, const ActivationForward& a)
    {
        switch (kind)
        {
        case kNone:
            return forward<kNone, DT, false>(s, a);
        case kSigmoid:
            return forward<kSigmoid, DT>(s, a);
        case kTanh:
            return forward<kTanh, DT>(s, a);
        case kRelu:
            return forward<kRelu, DT>(s, a);
        case kGelu:
            return forward<kGelu, DT>(s, a);
        case kSilu:
            return forward<kSilu, DT>(s, a);
        }
        return hipErrorInvalidValue;
    }
};
template <int DT>
struct Backward
{
    static hipError_t run(hipStream_t s, int kind, const ActivationBackward& a)
    {
        switch (kind)
        {
        case kSigmoid:
            return backward<kSigmoid, DT>(s, a);
        case kTanh:
            return backward<kTanh, DT>(s, a);
        case kRelu:
            return backward<kRelu, DT>(s, a);
        case kGelu:
            return backward<kGelu, DT>(s, a);
        case kSilu:
            return backward<kSilu, DT>(s, a);
        }
        return hipErrorInvalidValue;
    }
};
template <int DT>
struct Load8
{
    static hipError_t run(hipStream_t s, const void* saved, size_t rows, size_t cols, void* out, int64_t stride)
    {
        const RowGrid g = row_grid(rows, cols);
        load8_kernel<DT><<<row_blocks(g), kThreads, 0, s>>>(saved, out, stride, g);
        return hipGetLastError();
    }
};

} // namespace

size_t row_workgroups(size_t rows, size_t cols)
{
    const RowGrid g = row_grid(0, cols);
    return ceil_div(rows, (size_t) (kThreads >> g.lanes_log)) * g.chunks;
}

hipError_t launch_activation_forward(hipStream_t s, int kind, int dtype, const ActivationForward& a)
{
    return by_dtype<Forward>(dtype, s, kind, a);
}
hipError_t launch_activation_backward(hipStream_t s, int kind, int dtype, const ActivationBackward& a)
{
    return by_dtype<Backward>(dtype, s, kind, a);
}
hipError_t launch_load8(hipStream_t s, int dtype, const void* saved, size_t rows, size_t cols, void* out, int64_t out_stride)
{
    return by_dtype<Load8>(dtype, s, saved, rows, cols, out, out_stride);
}

} // namespace lowbit
} // namespace cntkq
