// The end of one block and the start of the next: h = x + scale gate post(y), n = pre(h), and its gradients.
//
// With r = 1 / sqrt(mean(x^2) + eps), a norm is x r w, and its gradient for an upstream d is
//     dx = r w d - (x r) c,  c = r^2 / dim sum(w d x),    dw = sum over rows of d x r.
// (r^3 is no float32 for rows of size 1e13, or 1e-13 without an eps. r sum / dim is of w d's size for any x, so c is formed as
// that times r: see projection().)
// So a row needs, forward, sum y^2 then sum h^2, and backward sum h^2, sum w dn h and sum y^2 together, then (from
// g = dh + r_h w dn - h r_h c_h) sum w gate scale g y. All sums are float32, each thread's terms in column order, then the
// threads of a wave and the waves of a workgroup in a fixed tree: a row's bits depend on the row alone.
//
// Bound: HBM, each row array read and written once. 8192 x 2304 in bfloat16: forward 31.7 us, 4.8 TB/s; gradients 68 us, 3.3 TB/s,
// where two sums in a row over the workgroup leave gaps that its two or three workgroups on a CU do not fill (8192 x 4096: 87 us,
// 4.6 TB/s). 4099 x 2048 in float32 with a channel gate: 49 us, 4.1 TB/s. Gradients of rows that are more than a thread's registers
// are far from it: 16-bit rows of 8193 to 16384 elements (121 to 127 registers in scratch memory with a norm before the next
// block; 4096 x 12288: 596 us, 1.0 TB/s, where 4096 x 8192 has 3.6), rows of 4097 to 8192 that are not whole 16-byte chunks (56 to
// 62; 4096 x 6001: 306 us, 1.0 TB/s), and longer ones, which are read once for each sum (4096 x 20000: 1.46 ms, 0.7 TB/s).
#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "dllm_hip.h"
#include "element.h"
#include "lds_copy.h"
#include "workspace.h"

using namespace dllm_hip;

namespace {

struct NormArgs {
    const void *x, *y, *gate;  // x: the residual stream (forward), h (backward)
    const float *post_weight, *pre_weight;
    const void *dh, *dn;
    void *h, *n;             // forward outputs
    void *dx, *dy, *dgate;   // backward outputs
    float *stats;            // [rows][4]: r_h, c_h, r_y, c_y
    float *partial;          // [3][chunks][dim]: gate, post, pre
    int64_t rows, dim;
    int post, pre, gate_kind;
    float offset;  // 1 with unit_offset
    float eps, scale, inv_dim;
    int64_t chunk_rows;
    int sums;  // bit 0: dgate, 1: dpost_weight, 2: dpre_weight
};

// The sum of a wave's 64 values, in every lane: rows of 16 lanes by shifts, then across the rows (data-parallel primitives:
// no trip through LDS).
template <int kControl>
__device__ __forceinline__ float shifted(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += shifted<0x111>(v);  // row_shr 1, 2, 4, 8
    v += shifted<0x112>(v);
    v += shifted<0x114>(v);
    v += shifted<0x118>(v);
    v += shifted<0x142>(v);  // each row's last lane to the next row, then lane 31 to the upper half
    v += shifted<0x143>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Sums of a workgroup's values, the waves' added in wave order; every thread gets them. scratch: 16 * N floats.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* scratch) {
    const int wave = static_cast<int>(threadIdx.x) >> 6, waves = static_cast<int>(blockDim.x) >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if (waves == 1) return;
    __syncthreads();  // the scratch's readers of the last sum are done
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[wave * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float t = scratch[i];
        for (int w = 1; w < waves; ++w) t += scratch[w * N + i];
        v[i] = t;
    }
}

__device__ __forceinline__ float weight_at(const float* w, int64_t c, float offset) {
    return w ? offset + w[c] : 1.0f;
}

template <typename T>
__device__ __forceinline__ float gate_at(const NormArgs& a, int64_t row, int64_t c) {
    if (a.gate_kind == 0) return 1.0f;
    if (a.gate_kind == 1) return static_cast<const float*>(a.gate)[c];
    return static_cast<float>(static_cast<const T*>(a.gate)[row * a.dim + c]);
}

__device__ __forceinline__ float inverse_rms(float sum_squares, const NormArgs& a) {
    return 1.0f / sqrtf(sum_squares * a.inv_dim + a.eps);
}

// c of a norm's gradient from r and sum(w d x).
__device__ __forceinline__ float projection(float r, float sum, const NormArgs& a) { return r * sum * a.inv_dim * r; }

// ---- rows of any size and alignment: one workgroup per row, a pass over it for each sum ----

template <typename T>
__global__ __launch_bounds__(256) void forward_any_kernel(NormArgs a) {
    __shared__ float scratch[16];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.dim;
        const T* y = static_cast<const T*>(a.y) + row * a.dim;
        float ry = 1.0f, rh = 1.0f;
        if (a.post) {
            float s[1] = {0.0f};
            for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
                const float v = static_cast<float>(y[c]);
                s[0] = fmaf(v, v, s[0]);
            }
            block_sum(s, scratch);
            ry = inverse_rms(s[0], a);
        }
        auto new_h = [&](int64_t c) {
            float z = static_cast<float>(y[c]);
            if (a.post) z = z * ry * weight_at(a.post_weight, c, a.offset);
            return fmaf(a.scale, z * gate_at<T>(a, row, c), static_cast<float>(x[c]));
        };
        if (a.pre) {
            float s[1] = {0.0f};
            for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
                const float v = new_h(c);
                s[0] = fmaf(v, v, s[0]);
            }
            block_sum(s, scratch);
            rh = inverse_rms(s[0], a);
        }
        for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
            const float v = new_h(c);  // h may be x: read before it is written, by the same thread
            static_cast<T*>(a.h)[row * a.dim + c] = static_cast<T>(v);
            if (a.pre) static_cast<T*>(a.n)[row * a.dim + c] = static_cast<T>(v * rh * weight_at(a.pre_weight, c, a.offset));
        }
    }
}

// The gradient of h through its uses, and the parts of it that the post norm and the gate see, at one element.
template <typename T>
struct BackwardElement {
    float g, y, z, hat_y, w_post, gate, du;
    __device__ BackwardElement(const NormArgs& a, int64_t row, int64_t c, float rh, float ch, float ry) {
        const int64_t at = row * a.dim + c;
        g = a.dh ? static_cast<float>(static_cast<const T*>(a.dh)[at]) : 0.0f;
        if (a.pre)
            g += fmaf(rh * weight_at(a.pre_weight, c, a.offset), static_cast<float>(static_cast<const T*>(a.dn)[at]),
                      -(static_cast<float>(static_cast<const T*>(a.x)[at]) * rh * ch));
        y = static_cast<float>(static_cast<const T*>(a.y)[at]);
        hat_y = a.post ? y * ry : y;
        w_post = a.post ? weight_at(a.post_weight, c, a.offset) : 1.0f;
        z = hat_y * w_post;
        gate = gate_at<T>(a, row, c);
        du = a.scale * g * gate;
    }
};

template <typename T>
__global__ __launch_bounds__(256) void backward_stats_any_kernel(NormArgs a) {
    __shared__ float scratch[16];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* h = static_cast<const T*>(a.x) + row * a.dim;
        const T* y = static_cast<const T*>(a.y) + row * a.dim;
        float s[3] = {0.0f, 0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
            if (a.pre) {
                const float v = static_cast<float>(h[c]);
                s[0] = fmaf(v, v, s[0]);
                s[1] = fmaf(weight_at(a.pre_weight, c, a.offset) * static_cast<float>(static_cast<const T*>(a.dn)[row * a.dim + c]),
                            v, s[1]);
            }
            if (a.post) {
                const float v = static_cast<float>(y[c]);
                s[2] = fmaf(v, v, s[2]);
            }
        }
        block_sum(s, scratch);
        const float rh = a.pre ? inverse_rms(s[0], a) : 0.0f;
        const float ch = a.pre ? projection(rh, s[1], a) : 0.0f;
        const float ry = a.post ? inverse_rms(s[2], a) : 1.0f;
        float cy = 0.0f;
        if (a.post) {
            float u[1] = {0.0f};
            for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
                const BackwardElement<T> e(a, row, c, rh, ch, ry);
                u[0] = fmaf(e.du * e.w_post, e.y, u[0]);
            }
            block_sum(u, scratch);
            cy = projection(ry, u[0], a);
        }
        if (threadIdx.x == 0) {
            float* st = a.stats + row * 4;
            st[0] = rh, st[1] = ch, st[2] = ry, st[3] = cy;
        }
    }
}

// partial[k][chunk][c]: the sums over one chunk of rows, in row order.
template <typename T>
__global__ __launch_bounds__(256) void backward_columns_any_kernel(NormArgs a) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t chunk = blockIdx.y, chunks = gridDim.y;
    if (c >= a.dim) return;
    const int64_t end = std::min<int64_t>(a.rows, (chunk + 1) * a.chunk_rows);
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int64_t row = chunk * a.chunk_rows; row < end; ++row) {
        const float* st = a.stats + row * 4;
        const BackwardElement<T> e(a, row, c, st[0], st[1], st[2]);
        s[0] = fmaf(a.scale * e.g, e.z, s[0]);
        s[1] = fmaf(e.du, e.hat_y, s[1]);
        if (a.pre)
            s[2] = fmaf(static_cast<float>(static_cast<const T*>(a.dn)[row * a.dim + c]),
                        static_cast<float>(static_cast<const T*>(a.x)[row * a.dim + c]) * st[0], s[2]);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
        if (a.sums >> k & 1) a.partial[(k * chunks + chunk) * a.dim + c] = s[k];
}

template <typename T>
__global__ __launch_bounds__(256) void backward_rows_any_kernel(NormArgs a) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* st = a.stats + row * 4;
        for (int64_t c = threadIdx.x; c < a.dim; c += 256) {
            const BackwardElement<T> e(a, row, c, st[0], st[1], st[2]);
            const int64_t at = row * a.dim + c;
            if (a.dx) static_cast<T*>(a.dx)[at] = static_cast<T>(e.g);  // dx may be dh: read above by the same thread
            if (a.dgate && a.gate_kind == 2) static_cast<T*>(a.dgate)[at] = static_cast<T>(a.scale * e.g * e.z);
            if (a.dy) static_cast<T*>(a.dy)[at] = static_cast<T>(a.post ? fmaf(st[2] * e.w_post, e.du, -(e.hat_y * st[3])) : e.du);
        }
    }
}

// ---- rows of whole vectors, held in registers ----
//
// A workgroup has a row, a thread kVectors vectors of kWidth consecutive elements, blockDim vectors apart, so that a row is
// read once and its sums need one barrier each. kWidth is a 16-byte access, or 1 where rows or pointers are not whole ones.

template <typename T, int kWidth>
struct Vector {
    Pack<T, kWidth> raw;
    __device__ __forceinline__ void load(const void* array, int64_t at, bool in) {
        if (in) raw = *reinterpret_cast<const Pack<T, kWidth>*>(static_cast<const T*>(array) + at);
        else raw = Pack<T, kWidth>{};
    }
    // Without a branch: lanes outside read the row's first elements.
    __device__ __forceinline__ void load_all(const T* row, int64_t c) { raw = *reinterpret_cast<const Pack<T, kWidth>*>(row + c); }
    __device__ __forceinline__ void keep_if(bool in) {
        constexpr int kWords = (kWidth * sizeof(T) + 3) / 4;
        if constexpr (kWidth * sizeof(T) % 4 == 0) {
            union {
                Pack<T, kWidth> p;
                uint32_t w[kWords];
            } u{raw};
#pragma unroll
            for (int i = 0; i < kWords; ++i) u.w[i] = in ? u.w[i] : 0u;
            raw = u.p;
        } else {
            raw.v[0] = in ? raw.v[0] : static_cast<T>(0.0f);
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return static_cast<float>(raw.v[i]); }
};

// A float32 parameter at kWidth channels: offset + value, or ones where there is none.
template <int kWidth>
__device__ __forceinline__ void load_weight(const float* w, int64_t c, bool in, float offset, float (&out)[kWidth]) {
#pragma unroll
    for (int i = 0; i < kWidth; ++i) out[i] = w ? 0.0f : 1.0f;
    if (!w || !in) return;
    constexpr int kPart = kWidth < 4 ? kWidth : 4;
#pragma unroll
    for (int p = 0; p < kWidth / kPart; ++p) {
        float v[kPart];
        load_as_float<float, kPart>(w + c + p * kPart, v);
#pragma unroll
        for (int i = 0; i < kPart; ++i) out[p * kPart + i] = offset + v[i];
    }
}

// Sums over the workgroup with one barrier: the caller alternates between two scratch areas.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* scratch) {
    const int wave = static_cast<int>(threadIdx.x) >> 6, waves = static_cast<int>(blockDim.x) >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if (waves == 1) return;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[wave * N + i] = v[i];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = scratch[i];
    for (int w = 1; w < waves; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += scratch[w * N + i];
}

constexpr int kRowThreads = 512;  // at most, of a row

// Whether two rows of `arrays` arrays fit a thread's registers: the next one's loads are then in flight while the sums of
// this one are formed. They are loaded without branches, or a wait for one row would be a wait for both.
template <typename T, int kWidth, int kVectors, int kArrays>
constexpr bool kRowAhead = kArrays * kVectors * (kWidth * sizeof(T) > 4 ? kWidth * sizeof(T) / 4 : 1) <= 40;

template <typename T, int kWidth, int kVectors, bool kPre, bool kElementGate>
__global__ __launch_bounds__(kRowThreads) void forward_kernel(NormArgs a) {
    constexpr bool kAhead = kRowAhead<T, kWidth, kVectors, 3>;
    constexpr bool kHeld = kVectors * kWidth <= 8;  // parameters
    __shared__ float first_scratch[16], second_scratch[16];
    int64_t c[kVectors];
    bool in[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
        c[k] = (static_cast<int64_t>(k) * blockDim.x + threadIdx.x) * kWidth;
        in[k] = c[k] < a.dim;
    }
    struct Row {
        Vector<T, kWidth> x[kVectors], y[kVectors], gate[kVectors];
    };
    auto load = [&](Row& to, int64_t row) {
        const int64_t at = std::min(row, a.rows - 1) * a.dim;
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            const int64_t column = in[k] ? c[k] : 0;
            to.x[k].load_all(static_cast<const T*>(a.x) + at, column);
            to.y[k].load_all(static_cast<const T*>(a.y) + at, column);
            if constexpr (kElementGate) to.gate[k].load_all(static_cast<const T*>(a.gate) + at, column);
        }
    };
    auto mask = [&](Row& r) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            r.x[k].keep_if(in[k]), r.y[k].keep_if(in[k]);
            if constexpr (kElementGate) r.gate[k].keep_if(in[k]);
        }
    };
    auto from_memory = [&](int which, int k, float (&w)[kWidth]) {
        if (which == 0) load_weight<kWidth>(a.post ? a.post_weight : nullptr, c[k], in[k], a.offset, w);
        if (which == 1) load_weight<kWidth>(kPre ? a.pre_weight : nullptr, c[k], in[k], a.offset, w);
        if (which == 2) load_weight<kWidth>(a.gate_kind == 1 ? static_cast<const float*>(a.gate) : nullptr, c[k], in[k], 0.0f, w);
    };
    float held[3][kHeld ? kVectors : 1][kWidth];
    if constexpr (kHeld)
#pragma unroll
        for (int k = 0; k < kVectors; ++k)
#pragma unroll
            for (int which = 0; which < 3; ++which) from_memory(which, k, held[which][k]);
    auto parameter = [&](int which, int k, float (&w)[kWidth]) {
        if constexpr (kHeld) {
#pragma unroll
            for (int i = 0; i < kWidth; ++i) w[i] = held[which][k][i];
        } else {
            from_memory(which, k, w);
        }
    };

    Row now, next;
    if constexpr (kAhead) load(now, blockIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        load(kAhead ? next : now, kAhead ? row + gridDim.x : row);
        mask(now);
        float s[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < kVectors; ++k)
#pragma unroll
            for (int i = 0; i < kWidth; ++i) s[0] = fmaf(now.y[k][i], now.y[k][i], s[0]);
        if (a.post || kPre) row_sum(s, first_scratch);  // (its barrier frees the second sum's scratch)
        const float ry = a.post ? inverse_rms(s[0], a) : 1.0f;
        float h[kVectors][kWidth], t[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            float w[kWidth], g[kWidth];
            parameter(0, k, w);
            parameter(2, k, g);
#pragma unroll
            for (int i = 0; i < kWidth; ++i) {
                float gated = g[i];
                if constexpr (kElementGate) gated = now.gate[k][i];
                h[k][i] = fmaf(a.scale, now.y[k][i] * ry * w[i] * gated, now.x[k][i]);
                t[0] = fmaf(h[k][i], h[k][i], t[0]);
            }
            if (in[k]) store_from_float<T, kWidth>(static_cast<T*>(a.h) + row * a.dim + c[k], h[k]);
        }
        if constexpr (kPre) {
            row_sum(t, second_scratch);
            const float rh = inverse_rms(t[0], a);
#pragma unroll
            for (int k = 0; k < kVectors; ++k) {
                float w[kWidth];
                parameter(1, k, w);
#pragma unroll
                for (int i = 0; i < kWidth; ++i) h[k][i] = h[k][i] * rh * w[i];
                if (in[k]) store_from_float<T, kWidth>(static_cast<T*>(a.n) + row * a.dim + c[k], h[k]);
            }
        } else {
            lds_barrier();  // frees the first sum's scratch
        }
        if constexpr (kAhead) now = next;
    }
}

// The gradients of one row after another, the next row's loads in flight while the sums of this one are formed (where two
// rows fit the registers); a thread keeps its columns' sums of the gate's and the weights' gradients, which are added over
// the workgroups afterwards. kPre: a norm before the next block; kElementGate: a gate for each element.
template <typename T, int kWidth, int kVectors, bool kPre, bool kElementGate>
__global__ __launch_bounds__(kRowThreads) void backward_kernel(NormArgs a) {
    constexpr bool kAhead = kRowAhead<T, kWidth, kVectors, 5>;
    __shared__ float first_scratch[3 * 16], second_scratch[16];
    float sums[3][kVectors][kWidth] = {};
    int64_t c[kVectors];
    bool in[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
        c[k] = (static_cast<int64_t>(k) * blockDim.x + threadIdx.x) * kWidth;
        in[k] = c[k] < a.dim;
    }
    struct Row {
        Vector<T, kWidth> h[kVectors], y[kVectors], dh[kVectors], dn[kVectors], gate[kVectors];
    };
    const T* const dh_array = static_cast<const T*>(a.dh ? a.dh : a.y);  // something to load where there is none
    auto load = [&](Row& to, int64_t row) {
        const int64_t at = std::min(row, a.rows - 1) * a.dim;
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            const int64_t column = in[k] ? c[k] : 0;
            if constexpr (kPre) to.h[k].load_all(static_cast<const T*>(a.x) + at, column);
            if constexpr (kPre) to.dn[k].load_all(static_cast<const T*>(a.dn) + at, column);
            to.y[k].load_all(static_cast<const T*>(a.y) + at, column);
            to.dh[k].load_all(dh_array + at, column);
            if constexpr (kElementGate) to.gate[k].load_all(static_cast<const T*>(a.gate) + at, column);
        }
    };
    auto mask = [&](Row& r) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            if constexpr (kPre) r.h[k].keep_if(in[k]), r.dn[k].keep_if(in[k]);
            r.y[k].keep_if(in[k]);
            r.dh[k].keep_if(in[k] && a.dh);
            if constexpr (kElementGate) r.gate[k].keep_if(in[k]);
        }
    };
    // Parameters stay in registers where they are few, else in LDS (each thread its own): a load from memory here would be
    // waited for together with the next row's. (8192 rows of bfloat16, eight elements to a thread, registers and LDS: 4096 wide
    // 87 and 91 us, 2304 wide 70 and 64, 896 wide 25 and 28.)
    constexpr bool kHeld = kVectors * kWidth <= 8;
    extern __shared__ __attribute__((aligned(16))) float parameter_lds[];  // [3][blockDim * kVectors * kWidth], or nothing
    float held[3][kHeld ? kVectors : 1][kWidth];
    const int area = static_cast<int>(blockDim.x) * kVectors * kWidth;
    auto in_lds = [&](int which, int k) { return parameter_lds + which * area + static_cast<int>(c[k]); };
    auto from_memory = [&](int k, float (&post)[kWidth], float (&pre)[kWidth], float (&gate)[kWidth]) {
        load_weight<kWidth>(a.post ? a.post_weight : nullptr, c[k], in[k], a.offset, post);
        load_weight<kWidth>(kPre ? a.pre_weight : nullptr, c[k], in[k], a.offset, pre);
        load_weight<kWidth>(a.gate_kind == 1 ? static_cast<const float*>(a.gate) : nullptr, c[k], in[k], 0.0f, gate);
    };
    if constexpr (kHeld) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) from_memory(k, held[0][k], held[1][k], held[2][k]);
    } else if constexpr (kAhead) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            float w[3][kWidth];
            from_memory(k, w[0], w[1], w[2]);
#pragma unroll
            for (int which = 0; which < 3; ++which)
#pragma unroll
                for (int i = 0; i < kWidth; ++i) in_lds(which, k)[i] = w[which][i];
        }
    }
    auto parameters = [&](int k, float (&post)[kWidth], float (&pre)[kWidth], float (&gate)[kWidth]) {
        if constexpr (kHeld || kAhead) {
#pragma unroll
            for (int i = 0; i < kWidth; ++i) {
                post[i] = kHeld ? held[0][kHeld ? k : 0][i] : in_lds(0, k)[i];
                pre[i] = kHeld ? held[1][kHeld ? k : 0][i] : in_lds(1, k)[i];
                gate[i] = kHeld ? held[2][kHeld ? k : 0][i] : in_lds(2, k)[i];
            }
        } else {
            from_memory(k, post, pre, gate);
        }
    };

    Row now, next;
    if constexpr (kAhead) load(now, blockIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        load(kAhead ? next : now, kAhead ? row + gridDim.x : row);
        mask(now);
        float s[kPre ? 3 : 1] = {};
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            float post[kWidth], pre[kWidth], gate[kWidth];
            parameters(k, post, pre, gate);
#pragma unroll
            for (int i = 0; i < kWidth; ++i) {
                const float y = now.y[k][i];
                s[0] = fmaf(y, y, s[0]);
                if constexpr (kPre) {
                    const float h = now.h[k][i];
                    s[1] = fmaf(h, h, s[1]);
                    s[2] = fmaf(pre[i] * now.dn[k][i], h, s[2]);
                }
            }
        }
        row_sum(s, first_scratch);
        const float ry = a.post ? inverse_rms(s[0], a) : 1.0f;
        float rh = 0.0f, ch = 0.0f;
        if constexpr (kPre) {
            rh = inverse_rms(s[1], a);
            ch = projection(rh, s[2], a);
        }
        float du[kVectors][kWidth], u[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
            float post[kWidth], pre[kWidth], gate[kWidth], g[kWidth], dgate[kWidth];
            parameters(k, post, pre, gate);
#pragma unroll
            for (int i = 0; i < kWidth; ++i) {
                const float y = now.y[k][i], hat = y * ry;
                g[i] = now.dh[k][i];
                if constexpr (kPre) {
                    const float h = now.h[k][i], dn = now.dn[k][i];
                    const float hat_h = h * rh;
                    g[i] += fmaf(rh * pre[i], dn, -(hat_h * ch));
                    sums[2][k][i] = fmaf(dn, hat_h, sums[2][k][i]);
                }
                const float dz = a.scale * g[i];
                float gated = gate[i];
                if constexpr (kElementGate) gated = now.gate[k][i];
                dgate[i] = dz * (hat * post[i]);
                du[k][i] = dz * gated;
                u[0] = fmaf(du[k][i] * post[i], y, u[0]);
                sums[0][k][i] += dgate[i];
                sums[1][k][i] = fmaf(du[k][i], hat, sums[1][k][i]);
            }
            const int64_t at = row * a.dim + c[k];
            if (a.dx && in[k]) store_from_float<T, kWidth>(static_cast<T*>(a.dx) + at, g);
            if constexpr (kElementGate)
                if (a.dgate && in[k]) store_from_float<T, kWidth>(static_cast<T*>(a.dgate) + at, dgate);
        }
        // (also where no dy is asked for: the barrier of this sum frees the first one's scratch)
        row_sum(u, second_scratch);
        const float cy = a.post ? projection(ry, u[0], a) : 0.0f;
        if (a.dy)
#pragma unroll
            for (int k = 0; k < kVectors; ++k) {
                float post[kWidth], pre[kWidth], gate[kWidth], dy[kWidth];
                parameters(k, post, pre, gate);
#pragma unroll
                for (int i = 0; i < kWidth; ++i)
                    dy[i] = a.post ? fmaf(ry * post[i], du[k][i], -(now.y[k][i] * ry * cy)) : du[k][i];
                if (in[k]) store_from_float<T, kWidth>(static_cast<T*>(a.dy) + row * a.dim + c[k], dy);
            }
        if constexpr (kAhead) now = next;
    }
#pragma unroll
    for (int which = 0; which < 3; ++which)
        if (a.sums >> which & 1)
#pragma unroll
            for (int k = 0; k < kVectors; ++k)
                if (in[k]) {
                    float* to = a.partial + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * a.dim + c[k];
                    if constexpr (kWidth == 1) {
                        to[0] = sums[which][k][0];
                    } else {
#pragma unroll
                        for (int i = 0; i < kWidth; i += 4) store_from_float<float, 4>(to + i, *reinterpret_cast<float(*)[4]>(&sums[which][k][i]));
                    }
                }
}

// out[c] = the chunks' sums of column c: 64 threads take every 64th chunk in order, then are added in a fixed tree. 16 columns
// (a 64-byte piece of a row of sums) to a workgroup, so that a few thousand columns fill the CUs.
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float* __restrict__ partial, float* dgate,
                                                             float* dpost, float* dpre, int64_t dim, int64_t chunks) {
    __shared__ float part[16][16];
    float* const out = blockIdx.y == 0 ? dgate : blockIdx.y == 1 ? dpost : dpre;
    if (!out) return;
    const int col = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + col;
    const float* p = partial + static_cast<int64_t>(blockIdx.y) * chunks * dim;
    float s = 0.0f;
    if (c < dim) {
#pragma unroll 8
        for (int64_t k = threadIdx.x >> 4; k < chunks; k += 64) s += p[k * dim + c];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 63) < 16) part[wave][col] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= dim) return;
    s = part[0][col];
    for (int r = 1; r < 16; ++r) s += part[r][col];
    out[c] = s;
}

constexpr int64_t kMaxGrid = 1 << 16;  // rows beyond it are taken in turn

int64_t any_chunk_rows(int64_t rows) { return std::max<int64_t>(64, ceil_div(rows, 1024)); }

// Workgroups that the rows are dealt to, each with the next row's loads in flight: four to a CU forward and two backward, where
// more would add column sums to be written and read again; more of the smaller ones that rows below 2048 elements make.
// Measured for 8192 x 2304 bfloat16, forward: 34.7 us with 512, 31.7 with 1024, 34.1 with 2048, 38.1 with one row each;
// backward: 69 us with 512, 80 with 768. 16384 rows of 64, forward: 22.2 us with 512, 11.7 with 1024, 7.9 with 2048.
int64_t row_groups(int64_t rows, int64_t dim, int64_t most) { return std::min(rows, most * 2048 / std::clamp<int64_t>(dim, 512, 2048)); }
constexpr int64_t kForwardGroups = 1024, kBackwardGroups = 512;

struct BackwardLayout {
    int64_t chunks;
    size_t stats, partial, bytes;
};

BackwardLayout backward_layout(const dllm_hip_residual_norm_shape& sh) {
    BackwardLayout b;
    Layout l;
    b.stats = static_cast<size_t>(sh.rows) * 4;
    b.chunks = static_cast<int64_t>(ceil_div(sh.rows, any_chunk_rows(sh.rows)));
    b.partial = static_cast<size_t>(3 * std::max(b.chunks, row_groups(sh.rows, sh.dim, kBackwardGroups)) * sh.dim);
    l.add<float>(b.stats);
    l.add<float>(b.partial);
    b.bytes = l.bytes;
    return b;
}

// Threads and vectors of a row of `vectors` vectors: the fewest vectors to a thread that `most` threads can take; 0 where
// `deepest` to a thread are not enough.
struct RowShape {
    int threads, each;
};
RowShape row_shape(int64_t vectors, int most, int deepest) {
    for (int each = 1; each <= deepest; each *= 2) {
        const int64_t threads = static_cast<int64_t>(round_up(ceil_div(vectors, each), 64));
        if (threads <= most) return {static_cast<int>(threads), each};
    }
    return {0, 0};
}

int check_shape(const dllm_hip_residual_norm_shape* sh) {
    DLLM_REQUIRE(sh != nullptr, "null shape");
    DLLM_REQUIRE(sh->dtype >= 0 && sh->dtype <= 2, "dtype must be float32 (0), bfloat16 (1) or float16 (2)");
    DLLM_REQUIRE(sh->rows >= 0 && sh->rows < (int64_t{1} << 31), "rows must be in [0, 2^31)");
    DLLM_REQUIRE(sh->dim >= 1 && sh->dim <= (1 << 20), "dim must be in [1, 2^20]");
    DLLM_REQUIRE(sh->norm_placement >= 0 && sh->norm_placement <= 2, "norm_placement must be pre (0), post (1) or both (2)");
    DLLM_REQUIRE(sh->gate >= 0 && sh->gate <= 2, "gate must be none (0), per channel (1) or per element (2)");
    DLLM_REQUIRE(sh->eps >= 0.0, "eps must not be negative");
    return kOk;
}

NormArgs arguments(const dllm_hip_residual_norm_shape& sh) {
    NormArgs a{};
    a.rows = sh.rows;
    a.dim = sh.dim;
    a.post = sh.norm_placement != 0;
    a.pre = sh.norm_placement != 1;
    a.gate_kind = static_cast<int>(sh.gate);
    a.offset = sh.unit_offset ? 1.0f : 0.0f;
    a.eps = static_cast<float>(sh.eps);
    a.scale = static_cast<float>(sh.residual_scale);
    a.inv_dim = 1.0f / static_cast<float>(sh.dim);
    return a;
}

template <typename T, int kWidth, int kVectors>
void launch_forward_vectors(const NormArgs& a, int threads, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(row_groups(a.rows, a.dim, kForwardGroups));
    if (a.pre && a.gate_kind == 2)
        forward_kernel<T, kWidth, kVectors, true, true><<<grid, threads, 0, stream>>>(a);
    else if (a.pre)
        forward_kernel<T, kWidth, kVectors, true, false><<<grid, threads, 0, stream>>>(a);
    else if (a.gate_kind == 2)
        forward_kernel<T, kWidth, kVectors, false, true><<<grid, threads, 0, stream>>>(a);
    else
        forward_kernel<T, kWidth, kVectors, false, false><<<grid, threads, 0, stream>>>(a);
}

// The rows in registers; false where they are too long for it.
template <typename T, int kWidth>
bool launch_forward_rows(const NormArgs& a, hipStream_t stream) {
    const RowShape r = row_shape(a.dim / kWidth, kRowThreads, kWidth == 1 ? 16 : 4);
    if (r.each == 1) launch_forward_vectors<T, kWidth, 1>(a, r.threads, stream);
    if (r.each == 2) launch_forward_vectors<T, kWidth, 2>(a, r.threads, stream);
    if (r.each == 4) launch_forward_vectors<T, kWidth, 4>(a, r.threads, stream);
    if constexpr (kWidth == 1) {
        if (r.each == 8) launch_forward_vectors<T, 1, 8>(a, r.threads, stream);
        if (r.each == 16) launch_forward_vectors<T, 1, 16>(a, r.threads, stream);
    }
    return r.each != 0;
}

template <typename T>
int launch_forward(const NormArgs& a, bool whole, hipStream_t stream) {
    const bool done = whole ? launch_forward_rows<T, kChunk<T>>(a, stream) : launch_forward_rows<T, 1>(a, stream);
    if (!done) forward_any_kernel<T><<<static_cast<unsigned>(std::min(a.rows, kMaxGrid)), 256, 0, stream>>>(a);
    return check_launch("residual_norm");
}

template <typename T, int kWidth, int kVectors, bool kPre, bool kElementGate>
int launch_backward_kind(const NormArgs& a, dim3 grid, int threads, hipStream_t stream) {
    const bool lds = kRowAhead<T, kWidth, kVectors, 5> && kVectors * kWidth > 8;
    const int bytes = lds ? 3 * threads * kVectors * kWidth * 4 : 0;
    const auto kernel = backward_kernel<T, kWidth, kVectors, kPre, kElementGate>;
    if (bytes > 60 * 1024)
        DLLM_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
                           "residual_norm_backward"));
    kernel<<<grid, threads, bytes, stream>>>(a);
    return check_launch("residual_norm_backward");
}

template <typename T, int kWidth, int kVectors>
int launch_backward_vectors(const NormArgs& a, dim3 grid, int threads, hipStream_t stream) {
    if (a.pre && a.gate_kind == 2) return launch_backward_kind<T, kWidth, kVectors, true, true>(a, grid, threads, stream);
    if (a.pre) return launch_backward_kind<T, kWidth, kVectors, true, false>(a, grid, threads, stream);
    if (a.gate_kind == 2) return launch_backward_kind<T, kWidth, kVectors, false, true>(a, grid, threads, stream);
    return launch_backward_kind<T, kWidth, kVectors, false, false>(a, grid, threads, stream);
}

// The rows in registers, with `done`; not where they are too long for it.
template <typename T, int kWidth>
int launch_backward_rows(const NormArgs& a, unsigned groups, bool& done, hipStream_t stream) {
    const RowShape r = row_shape(a.dim / kWidth, kRowThreads, kWidth == 1 ? 16 : 4);
    done = r.each != 0;
    switch (r.each) {
        case 1: return launch_backward_vectors<T, kWidth, 1>(a, groups, r.threads, stream);
        case 2: return launch_backward_vectors<T, kWidth, 2>(a, groups, r.threads, stream);
        case 4: return launch_backward_vectors<T, kWidth, 4>(a, groups, r.threads, stream);
    }
    if constexpr (kWidth == 1) {
        if (r.each == 8) return launch_backward_vectors<T, 1, 8>(a, groups, r.threads, stream);
        if (r.each == 16) return launch_backward_vectors<T, 1, 16>(a, groups, r.threads, stream);
    }
    return kOk;
}

template <typename T>
int launch_backward(const NormArgs& a, bool whole, int64_t chunks, float* dpost, float* dpre, hipStream_t stream) {
    const unsigned groups = static_cast<unsigned>(row_groups(a.rows, a.dim, kBackwardGroups));
    const unsigned rows = static_cast<unsigned>(std::min(a.rows, kMaxGrid));
    bool done = false;
    if (whole)
        DLLM_TRY((launch_backward_rows<T, kChunk<T>>(a, groups, done, stream)));
    else
        DLLM_TRY((launch_backward_rows<T, 1>(a, groups, done, stream)));
    if (!done) backward_stats_any_kernel<T><<<rows, 256, 0, stream>>>(a);
    if (!done && a.sums)
        backward_columns_any_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(a.dim, 256)), static_cast<unsigned>(chunks)), 256, 0, stream>>>(a);
    if (a.sums)
        column_reduce_kernel<<<dim3(static_cast<unsigned>(ceil_div(a.dim, 16)), 3), 1024, 0, stream>>>(
            a.partial, a.sums & 1 ? static_cast<float*>(a.dgate) : nullptr, dpost, dpre, a.dim, done ? groups : chunks);
    // after the column sums: dx may be dh, which they read
    if (!done && (a.dx || a.dy || (a.dgate && a.gate_kind == 2))) backward_rows_any_kernel<T><<<rows, 256, 0, stream>>>(a);
    return check_launch("residual_norm_backward");
}

// Rows and pointers of whole 16-byte vectors.
bool whole_vectors(const NormArgs& a, size_t size, std::initializer_list<const void*> arrays) {
    bool whole = a.dim % static_cast<int64_t>(16 / size) == 0;
    for (const void* p : arrays) whole = whole && aligned_to(p, 16);
    return whole;
}

}  // namespace

extern "C" {

int dllm_hip_residual_norm(const dllm_hip_residual_norm_shape* sh, const void* x, const void* y, const void* gate,
                           const float* post_weight, const float* pre_weight, void* h, void* n, void* stream) {
    DLLM_TRY(check_shape(sh));
    if (sh->rows == 0) return kOk;
    NormArgs a = arguments(*sh);
    DLLM_REQUIRE(x && y && h && (n || !a.pre) && (gate || a.gate_kind == 0), "null x, y, gate, h or n");
    const size_t size = element_bytes(sh->dtype);
    DLLM_REQUIRE(aligned_to(x, size) && aligned_to(y, size) && aligned_to(h, size) && aligned_to(n, size) &&
                     aligned_to(gate, a.gate_kind == 1 ? 4 : size) && aligned_to(post_weight, 4) &&
                     aligned_to(pre_weight, 4),
                 "pointers must be aligned to the element");
    a.x = x, a.y = y, a.gate = gate, a.post_weight = post_weight, a.pre_weight = pre_weight, a.h = h, a.n = n;
    const bool whole = whole_vectors(a, size, {x, y, gate, post_weight, pre_weight, h, n});
    auto s = static_cast<hipStream_t>(stream);
    switch (sh->dtype) {
        case kFloat32: return launch_forward<float>(a, whole, s);
        case kBFloat16: return launch_forward<__bf16>(a, whole, s);
        default: return launch_forward<_Float16>(a, whole, s);
    }
}

size_t dllm_hip_residual_norm_backward_workspace(const dllm_hip_residual_norm_shape* sh) {
    return check_shape(sh) == kOk ? backward_layout(*sh).bytes : 0;
}

int dllm_hip_residual_norm_backward(const dllm_hip_residual_norm_shape* sh, const void* h, const void* y,
                                    const void* gate, const float* post_weight, const float* pre_weight,
                                    const void* dh, const void* dn, void* dx, void* dy, void* dgate,
                                    float* dpost_weight, float* dpre_weight, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    DLLM_TRY(check_shape(sh));
    NormArgs a = arguments(*sh);
    DLLM_REQUIRE(a.gate_kind || !dgate, "dgate without a gate");
    DLLM_REQUIRE((a.post || !dpost_weight) && (a.pre || !dpre_weight), "a weight gradient of a norm that is not there");
    auto s = static_cast<hipStream_t>(stream);
    if (sh->rows == 0) {  // sums over no rows
        for (float* out : {a.gate_kind == 1 ? static_cast<float*>(dgate) : nullptr, dpost_weight, dpre_weight})
            if (out) column_reduce_kernel<<<dim3(static_cast<unsigned>(ceil_div(a.dim, 16))), 1024, 0, s>>>(nullptr, out, nullptr, nullptr, a.dim, 0);
        return check_launch("residual_norm_backward");
    }
    DLLM_REQUIRE((h || !a.pre) && y && (gate || a.gate_kind == 0) && (dn || !a.pre) && (dh || a.pre),
                 "null h, y, gate, dh or dn");
    const size_t size = element_bytes(sh->dtype);
    for (const void* p : {h, y, dh, dn, static_cast<const void*>(dx), static_cast<const void*>(dy)})
        DLLM_REQUIRE(aligned_to(p, size), "pointers must be aligned to the element");
    for (const void* p : {gate, static_cast<const void*>(dgate)})
        DLLM_REQUIRE(aligned_to(p, a.gate_kind == 1 ? 4 : size), "pointers must be aligned to the element");
    for (const float* p : {post_weight, pre_weight, static_cast<const float*>(dpost_weight), static_cast<const float*>(dpre_weight)})
        DLLM_REQUIRE(aligned_to(p, 4), "pointers must be aligned to the element");
    const BackwardLayout b = backward_layout(*sh);
    DLLM_REQUIRE(workspace && workspace_bytes >= b.bytes, "workspace too small for residual_norm_backward");
    DLLM_REQUIRE(aligned_to(workspace, 16), "the workspace must be aligned to 16 bytes");
    Carve c(workspace, workspace_bytes);
    a.stats = c.take<float>(b.stats);
    a.partial = c.take<float>(b.partial);
    a.x = h, a.y = y, a.gate = gate, a.post_weight = post_weight, a.pre_weight = pre_weight, a.dh = dh, a.dn = dn;
    a.dx = dx, a.dy = dy, a.dgate = dgate;
    a.chunk_rows = any_chunk_rows(sh->rows);
    a.sums = (a.gate_kind == 1 && dgate ? 1 : 0) | (dpost_weight ? 2 : 0) | (dpre_weight ? 4 : 0);
    const bool whole = whole_vectors(a, size, {h, y, gate, post_weight, pre_weight, dh, dn, dx, dy, dgate});
    switch (sh->dtype) {
        case kFloat32: return launch_backward<float>(a, whole, b.chunks, dpost_weight, dpre_weight, s);
        case kBFloat16: return launch_backward<__bf16>(a, whole, b.chunks, dpost_weight, dpre_weight, s);
        default: return launch_backward<_Float16>(a, whole, b.chunks, dpost_weight, dpre_weight, s);
    }
}

}  // extern "C"
