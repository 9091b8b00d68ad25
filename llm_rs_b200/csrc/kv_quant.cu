// Scaled rotary positions and the 8-bit KV cache: rotation from a frequency table, quantisation of keys
// and values as they are written to their slots, rows read back.
//
// Cache: a pool of E4M3 codes, [kv_dim, slots], and one float32 scale per (slot, KV head), [slots, heads]
// (slots contiguous: the scales of one head at consecutive positions of a page are one run of memory for
// the attention that reads them).  value = code * scale with
//   scale = max(amax / 448, 2^-126)   over the head's values in float32, 448 the largest E4M3 number,
//   code  = E4M3, round to nearest even, of value / scale (IEEE division: the result is a definition, not an
//           approximation, so any implementation reproduces it bit for bit).
// 2^-126 keeps the division away from zero and from quotients of subnormal scales.  A head row with a
// value that is not finite is stored as scale NaN and codes 0: the codes of the cache are always finite, and
// attention, which applies the scales outside the matrix instructions, can leave such a position out by a
// select; a NaN code would get through a product with a weight of zero.
#include <cuda_fp8.h>

#include "kernels.h"
#include "llmrs_common.cuh"
#include "pipeline.cuh"

namespace llmrs {

namespace {

constexpr int RW_THREADS = 128;

// V consecutive elements between memory and float registers, in one access (V * sizeof(T) = 16, or one element).
template <typename T, int V> struct Chunk;
template <> struct Chunk<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void load(float *x, const __nv_bfloat16 *p) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Chunk<float, 4> {
    static __device__ __forceinline__ void load(float *x, const float *p) {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    }
    static __device__ __forceinline__ void store(float *p, const float *x) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
};
template <> struct Chunk<__nv_bfloat16, 1> {
    static __device__ __forceinline__ void load(float *x, const __nv_bfloat16 *p) { x[0] = __bfloat162float(*p); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) { *p = __float2bfloat16_rn(x[0]); }
};
template <> struct Chunk<float, 1> {
    static __device__ __forceinline__ void load(float *x, const float *p) { x[0] = *p; }
    static __device__ __forceinline__ void store(float *p, const float *x) { *p = x[0]; }
};

// V floats (already divided by their scale) -> V E4M3 codes.
template <int V> __device__ __forceinline__ void store_codes(uint8_t *p, const float *x) {
    if constexpr (V == 1) {
        *p = (uint8_t)__nv_cvt_float_to_fp8(x[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
            w[i] = lo | hi << 16;
        }
        if constexpr (V == 4) *reinterpret_cast<uint32_t *>(p) = w[0];
        else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
}

__device__ __forceinline__ void rotate(float &a, float &b, float2 t) {
    const float x0 = a, x1 = b;
    a = x0 * t.x - x1 * t.y;
    b = x0 * t.y + x1 * t.x;
}

// The rows of a token, in this order: nq heads of q, nk of k (both rotated), nv of v.  q goes to q_out, k to
// k_out (rope) or quantised to k_pool (write), v quantised to v_pool.  `lpr` lanes (a power of two) share
// a row; a lane owns up to ITER units of V pairs: in the half layout the elements V u .. V u + V and their
// partners rotary/2 further on, in the interleaved one 2 V consecutive elements, so both members of a pair are
// always in one thread, rotation in place is safe, and pair j of a unit has frequency V u + j in both.
// The cosines and sines of a token are formed once per CTA (one per thread, angle reduced in float64: at
// position 131072 a float32 angle has lost 7 of its fraction's bits) and shared by its 40 or so heads.
// HBM-bound: what is read and written is what the operation cannot do without.
template <typename T, int V, int ITER>
__global__ void __launch_bounds__(RW_THREADS) rope_write_kernel(const RopeWrite p) {
    pdl_prologue();
    __shared__ float2 cs[256];
    const int token = blockIdx.x;
    const int half = p.rotary / 2;
    if (p.nq + p.nk > 0) {
        const double pos = (double)p.positions[token];
        for (int i = threadIdx.x; i < half; i += RW_THREADS) {
            const double turns = pos * (double)p.inv_freq[i] * 0.15915494309189533577;      // 1 / (2 pi)
            float s, c;
            sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
            cs[i] = make_float2(c * p.magnitude, s * p.magnitude);
        }
        __syncthreads();
    }
    const int lpr = p.lanes_per_row, rpc = RW_THREADS / lpr;
    const int r = threadIdx.x / lpr, l = threadIdx.x % lpr;
    const int rows = p.nq + p.nk + p.nv, units = p.head_dim / (2 * V), rot_units = half / V;
    uint32_t slot = 0;
    bool to_cache = false;
    if (p.slots) {
        slot = p.slots[token];
        to_cache = slot < p.num_slots;
        if (!to_cache && slot != 0xFFFFFFFFu && threadIdx.x == 0) report_error(p.err, KERR_SLOT_RANGE);
    }
    for (int base = blockIdx.y * rpc; base < rows; base += gridDim.y * rpc) {       // the same trips for a whole warp
        const int row = base + r;
        const int which = row < p.nq ? 0 : row < p.nq + p.nk ? 1 : 2;
        const int head = which == 0 ? row : which == 1 ? row - p.nq : row - p.nq - p.nk;
        const int heads = which == 0 ? p.nq : which == 1 ? p.nk : p.nv;
        const size_t off = ((size_t)token * heads + head) * p.head_dim;
        const T *src = (const T *)(which == 0 ? p.q : which == 1 ? p.k : p.v);
        const bool quant = which == 2 || (which == 1 && p.k_pool);
        float x[ITER][2 * V];
        int at[ITER], bt[ITER];
        float amax = 0.0f;
        bool finite = true;
#pragma unroll
        for (int it = 0; it < ITER; it++) {
            const int u = l + it * lpr;
            const bool on = row < rows && u < units;
#pragma unroll
            for (int j = 0; j < 2 * V; j++) x[it][j] = 0.0f;
            const bool halves = p.split_half && u < rot_units && which != 2;
            at[it] = !on ? -1 : halves ? u * V : u * 2 * V;
            bt[it] = halves ? at[it] + half : at[it] + V;
            if (!on) continue;
            Chunk<T, V>::load(x[it], src + off + at[it]);
            Chunk<T, V>::load(x[it] + V, src + off + bt[it]);
            if (which != 2) {
                if (halves) {
#pragma unroll
                    for (int j = 0; j < V; j++) rotate(x[it][j], x[it][V + j], cs[u * V + j]);
                } else if (!p.split_half) {
#pragma unroll
                    for (int j = 0; j < V; j++)
                        if (u * V + j < half) rotate(x[it][2 * j], x[it][2 * j + 1], cs[u * V + j]);
                }
            }
            if (quant) {
#pragma unroll
                for (int j = 0; j < 2 * V; j++) {
                    amax = fmaxf(amax, fabsf(x[it][j]));
                    finite = finite && fabsf(x[it][j]) <= 3.402823466e38f;
                }
            } else {
                T *out = (T *)(which == 0 ? p.q_out : p.k_out);
                Chunk<T, V>::store(out + off + at[it], x[it]);
                Chunk<T, V>::store(out + off + bt[it], x[it] + V);
            }
        }
        if (!p.slots) continue;
        for (int o = lpr >> 1; o; o >>= 1) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            finite = __shfl_xor_sync(0xffffffffu, (int)finite, o) && finite;
        }
        if (!quant || row >= rows || !to_cache) continue;
        const float scale = fmaxf(amax / 448.0f, 1.17549435e-38f);
        uint8_t *pool = (which == 1 ? p.k_pool : p.v_pool) + ((size_t)slot * heads + head) * p.head_dim;
        float *scales = which == 1 ? p.k_scales : p.v_scales;
        if (l == 0) scales[(size_t)head * p.num_slots + slot] = finite ? scale : __int_as_float(0x7FC00000);
#pragma unroll
        for (int it = 0; it < ITER; it++) {
            if (at[it] < 0) continue;
#pragma unroll
            for (int j = 0; j < 2 * V; j++) x[it][j] = finite ? x[it][j] / scale : 0.0f;
            store_codes<V>(pool + at[it], x[it]);
            store_codes<V>(pool + bt[it], x[it] + V);
        }
    }
}

// Rows read back: out[c] = codes of slot indices[c], each head's times its scale.  A thread takes V codes of
// one head; one product and one rounding to the output type.
template <typename T, int V>
__global__ void __launch_bounds__(256)
gather_quant_kernel(T *__restrict__ out, const uint8_t *__restrict__ pool, const float *__restrict__ scales,
                    const uint32_t *__restrict__ indices, uint32_t kv_dim, uint32_t head_dim, uint32_t num_slots,
                    uint32_t rows, uint32_t *err) {
    pdl_prologue();
    const uint32_t units = kv_dim / V;
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (size_t)units * rows) return;
    const uint32_t row = (uint32_t)(i / units), d = (uint32_t)(i - (size_t)row * units) * V;
    const uint32_t slot = indices[row];
    if (slot >= num_slots) {                             // the row of out keeps what it held
        if (d == 0) report_error(err, KERR_SLOT_RANGE);
        return;
    }
    const uint8_t *src = pool + (size_t)slot * kv_dim + d;
    T *dst = out + (size_t)row * kv_dim + d;
    const float scale = scales[(size_t)(d / head_dim) * num_slots + slot];
    float x[V];
    if constexpr (V == 1) {
        x[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(*src, __NV_E4M3))) * scale;
        Chunk<T, 1>::store(dst, x);
    } else {
        uint32_t w[V / 4];
        if constexpr (V == 8) { const uint2 u = *reinterpret_cast<const uint2 *>(src); w[0] = u.x; w[1] = u.y; }
        else w[0] = *reinterpret_cast<const uint32_t *>(src);
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
            const __half2 h(__nv_cvt_fp8x2_to_halfraw2((uint16_t)(w[j / 2] >> (16 * (j & 1))), __NV_E4M3));
            const float2 f = __half22float2(h);
            x[2 * j] = f.x * scale;
            x[2 * j + 1] = f.y * scale;
        }
        Chunk<T, V>::store(dst, x);
    }
}

template <typename T, int VEC> cudaError_t rope_write(RopeWrite p, int tokens, int sm_count, cudaStream_t s, bool pdl) {
    const int hd = p.head_dim, half = p.rotary / 2;
    const bool vec = hd % (2 * VEC) == 0 && (!p.split_half || half % VEC == 0);
    const int v = vec ? VEC : 1, units = hd / (2 * v);
    int lpr = 1;
    while (lpr < 32 && lpr < units) lpr *= 2;
    p.lanes_per_row = lpr;
    const int rows = p.nq + p.nk + p.nv, rpc = RW_THREADS / lpr, most = (rows + rpc - 1) / rpc;
    const int want = (2 * sm_count + tokens - 1) / tokens;
    const dim3 grid((unsigned)tokens, (unsigned)(want < most ? want : most));
    if (vec) return launch_dependent(rope_write_kernel<T, VEC, 1>, grid, dim3(RW_THREADS), 0, s, pdl, p);
    return launch_dependent(rope_write_kernel<T, 1, 8>, grid, dim3(RW_THREADS), 0, s, pdl, p);
}

}  // namespace

cudaError_t launch_rope_write(const RopeWrite &p, int dtype, int tokens, int sm_count, cudaStream_t s, bool pdl) {
    if (tokens <= 0) return cudaSuccess;
    return dtype == DT_BF16 ? rope_write<__nv_bfloat16, 8>(p, tokens, sm_count, s, pdl)
                            : rope_write<float, 4>(p, tokens, sm_count, s, pdl);
}

cudaError_t launch_gather_quant(void *out, int dtype, const uint8_t *pool, const float *scales, const uint32_t *indices,
                                uint32_t kv_dim, uint32_t head_dim, uint32_t num_slots, uint32_t rows, uint32_t *err,
                                cudaStream_t s, bool pdl) {
    if (rows == 0) return cudaSuccess;
    const uint32_t vec = dtype == DT_BF16 ? 8 : 4;
    const bool ok = head_dim % vec == 0;
    const size_t n = (size_t)(kv_dim / (ok ? vec : 1)) * rows;
    const dim3 grid((unsigned)((n + 255) / 256));
#define LLMRS_GATHER(T, V) launch_dependent(gather_quant_kernel<T, V>, grid, dim3(256), 0, s, pdl, (T *)out, pool, scales, \
                                            indices, kv_dim, head_dim, num_slots, rows, err)
    if (dtype == DT_BF16) return ok ? LLMRS_GATHER(__nv_bfloat16, 8) : LLMRS_GATHER(__nv_bfloat16, 1);
    return ok ? LLMRS_GATHER(float, 4) : LLMRS_GATHER(float, 1);
#undef LLMRS_GATHER
}

}  // namespace llmrs
