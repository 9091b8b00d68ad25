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

// V consecutive elements between memory (Raw: one access) and float registers.
template <typename T, int V> struct Chunk;
template <> struct Chunk<__nv_bfloat16, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ void unpack(float *x, const Raw &u) {
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
    using Raw = float4;
    static __device__ __forceinline__ void unpack(float *x, const Raw &u) { x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; }
    static __device__ __forceinline__ void store(float *p, const float *x) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
};
template <> struct Chunk<__nv_bfloat16, 1> {
    using Raw = __nv_bfloat16;
    static __device__ __forceinline__ void unpack(float *x, const Raw &u) { x[0] = __bfloat162float(u); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) { *p = __float2bfloat16_rn(x[0]); }
};
template <> struct Chunk<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void unpack(float *x, const Raw &u) { x[0] = u; }
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
// HBM-bound: what is read and written is what the operation cannot do without.  So a thread asks for the units of
// PRE rows before anything else; the angles are formed while they are under way.
template <typename T, int V, int ITER, int PRE>
__global__ void __launch_bounds__(RW_THREADS) rope_write_kernel(const RopeWrite p) {
    using C = Chunk<T, V>;
    pdl_prologue();
    __shared__ float2 cs[128];
    const int token = blockIdx.x;
    const int half = p.rotary / 2;
    const int lpr = p.lanes_per_row, rpc = RW_THREADS / lpr, stride = gridDim.y * rpc;
    const int r = threadIdx.x / lpr, l = threadIdx.x % lpr;
    const int rows = p.nq + p.nk + p.nv, units = p.head_dim / (2 * V), rot_units = half / V;
    bool angles = p.nq + p.nk > 0, to_cache = false;
    uint32_t slot = 0;
    for (int base = blockIdx.y * rpc; base < rows; base += stride * PRE) {       // the same trips for a whole CTA
        typename C::Raw raw[PRE][ITER][2];
#pragma unroll
        for (int k = 0; k < PRE; k++) {
            const int row = base + k * stride + r;
            const int which = row < p.nq ? 0 : row < p.nq + p.nk ? 1 : 2;
            const int head = row - (which == 0 ? 0 : which == 1 ? p.nq : p.nq + p.nk), heads = which == 0 ? p.nq : which == 1 ? p.nk : p.nv;
            const T *src = (const T *)(which == 0 ? p.q : which == 1 ? p.k : p.v) + ((size_t)token * heads + head) * p.head_dim;
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int u = l + it * lpr;
                if (row >= rows || u >= units) continue;
                const bool halves = p.split_half && u < rot_units && which != 2;
                const int a = halves ? u * V : u * 2 * V, b = halves ? a + half : a + V;
                raw[k][it][0] = *reinterpret_cast<const typename C::Raw *>(src + a);
                raw[k][it][1] = *reinterpret_cast<const typename C::Raw *>(src + b);
            }
        }
        if (base == (int)blockIdx.y * rpc && p.slots) {
            slot = p.slots[token];
            to_cache = slot < p.num_slots;
            if (!to_cache && slot != 0xFFFFFFFFu && threadIdx.x == 0) report_error(p.err, KERR_SLOT_RANGE);
        }
        if (angles) {
            const double pos = (double)p.positions[token];
            for (int i = threadIdx.x; i < half; i += RW_THREADS) {
                const double turns = pos * (double)p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
                float s, c;
                sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
                cs[i] = make_float2(c * p.magnitude, s * p.magnitude);
            }
            __syncthreads();
            angles = false;
        }
#pragma unroll
        for (int k = 0; k < PRE; k++) {
            const int row = base + k * stride + r;
            if (base + k * stride >= rows) break;        // the whole CTA
            const int which = row < p.nq ? 0 : row < p.nq + p.nk ? 1 : 2;
            const int head = row - (which == 0 ? 0 : which == 1 ? p.nq : p.nq + p.nk), heads = which == 0 ? p.nq : which == 1 ? p.nk : p.nv;
            const bool quant = which == 2 || (which == 1 && p.k_pool);
            float x[ITER][2 * V];
            int at[ITER], bt[ITER];
            float amax = 0.0f;
            bool finite = true;
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int u = l + it * lpr;
                const bool on = row < rows && u < units;
                const bool halves = p.split_half && u < rot_units && which != 2;
                at[it] = !on ? -1 : halves ? u * V : u * 2 * V;
                bt[it] = halves ? at[it] + half : at[it] + V;
                if (!on) continue;
                C::unpack(x[it], raw[k][it][0]);
                C::unpack(x[it] + V, raw[k][it][1]);
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
                    T *out = (T *)(which == 0 ? p.q_out : p.k_out) + ((size_t)token * heads + head) * p.head_dim;
                    C::store(out + at[it], x[it]);
                    C::store(out + bt[it], x[it] + V);
                }
            }
            if (!p.slots || !__any_sync(0xffffffffu, quant && row < rows)) continue;
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
}

// Rows read back: out[c] = codes of slot indices[c], each head's times its scale; one product and one rounding.  A thread
// takes V codes of one head at a time (32 bytes of output, one store), of N units at once.  HBM-bound.
template <typename T, int V> __device__ __forceinline__ void store_row(T *p, const float *x) {
    if constexpr (V == 1) {
        Chunk<T, 1>::store(p, x);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (V == 8) {
                w[i] = __float_as_uint(x[i]);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                     "r"(w[6]), "r"(w[7])
                     : "memory");
    }
}
template <typename T, int V, int N>
__global__ void __launch_bounds__(256)
gather_quant_kernel(T *__restrict__ out, const uint8_t *__restrict__ pool, const float *__restrict__ scales,
                    const uint32_t *__restrict__ indices, uint32_t kv_dim, uint32_t head_dim, uint32_t num_slots,
                    uint32_t rows, uint32_t *err) {
    pdl_prologue();
    const uint32_t units = kv_dim / V;
    const size_t first = (size_t)blockIdx.x * (256 * N) + threadIdx.x, all = (size_t)units * rows;
    uint32_t d[N], row[N], slot[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const size_t i = first + k * 256;
        row[k] = i < all ? (uint32_t)(i / units) : 0xFFFFFFFFu;
        d[k] = (uint32_t)(i - (size_t)row[k] * units) * V;
        slot[k] = i < all ? indices[row[k]] : 0xFFFFFFFFu;
    }
    uint32_t w[N][V < 4 ? 1 : V / 4];
    float scale[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (slot[k] >= num_slots) continue;
        const uint8_t *src = pool + (size_t)slot[k] * kv_dim + d[k];
        scale[k] = scales[(size_t)(d[k] / head_dim) * num_slots + slot[k]];
        if constexpr (V == 16) { const uint4 u = *reinterpret_cast<const uint4 *>(src); w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w; }
        else if constexpr (V == 8) { const uint2 u = *reinterpret_cast<const uint2 *>(src); w[k][0] = u.x; w[k][1] = u.y; }
        else w[k][0] = *src;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (slot[k] >= num_slots) {                      // the row of out keeps what it held
            if (row[k] != 0xFFFFFFFFu && d[k] == 0) report_error(err, KERR_SLOT_RANGE);
            continue;
        }
        float x[V];
        if constexpr (V == 1) {
            x[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw((uint8_t)w[k][0], __NV_E4M3))) * scale[k];
        } else {
#pragma unroll
            for (int j = 0; j < V / 2; j++) {
                const __half2 h(__nv_cvt_fp8x2_to_halfraw2((uint16_t)(w[k][j / 2] >> (16 * (j & 1))), __NV_E4M3));
                const float2 f = __half22float2(h);
                x[2 * j] = f.x * scale[k];
                x[2 * j + 1] = f.y * scale[k];
            }
        }
        store_row<T, V>(out + (size_t)row[k] * kv_dim + d[k], x);
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
    if (vec) return launch_dependent(rope_write_kernel<T, VEC, 1, 3>, grid, dim3(RW_THREADS), 0, s, pdl, p);
    return launch_dependent(rope_write_kernel<T, 1, 4, 1>, grid, dim3(RW_THREADS), 0, s, pdl, p);
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
    const uint32_t vec = dtype == DT_BF16 ? 16 : 8;      // 32 bytes of output
    const bool ok = head_dim % vec == 0 && (uintptr_t)out % 32 == 0;
    const size_t n = (size_t)(kv_dim / (ok ? vec : 1)) * rows;
    constexpr int N = 4;
    // four units a thread once that still leaves every SM its share of warps; one each below
    const int per = n >= (size_t)4 * 256 * 148 * 4 ? N : 1;
    const dim3 grid((unsigned)((n + 256 * per - 1) / (256 * per)));
#define LLMRS_GATHER(T, V, K) launch_dependent(gather_quant_kernel<T, V, K>, grid, dim3(256), 0, s, pdl, (T *)out, pool, scales, \
                                               indices, kv_dim, head_dim, num_slots, rows, err)
    if (dtype == DT_BF16) {
        if (!ok) return per == N ? LLMRS_GATHER(__nv_bfloat16, 1, N) : LLMRS_GATHER(__nv_bfloat16, 1, 1);
        return per == N ? LLMRS_GATHER(__nv_bfloat16, 16, N) : LLMRS_GATHER(__nv_bfloat16, 16, 1);
    }
    if (!ok) return per == N ? LLMRS_GATHER(float, 1, N) : LLMRS_GATHER(float, 1, 1);
    return per == N ? LLMRS_GATHER(float, 8, N) : LLMRS_GATHER(float, 8, 1);
#undef LLMRS_GATHER
}

}  // namespace llmrs
