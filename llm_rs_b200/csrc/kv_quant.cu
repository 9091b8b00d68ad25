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

constexpr int RW_THREADS = 128, RW_TOKENS = 4;           // threads, most tokens of a CTA

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

// V floats -> V E4M3 codes of them times `f`, packed.
template <int V> __device__ __forceinline__ void codes_of(uint32_t (&w)[V < 4 ? 1 : V / 4], const float *x, float f) {
    if constexpr (V == 1) {
        w[0] = __nv_cvt_float_to_fp8(x[0] * f, __NV_SATFINITE, __NV_E4M3);
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * f, x[4 * i + 1] * f), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * f, x[4 * i + 3] * f), __NV_SATFINITE, __NV_E4M3);
            w[i] = __byte_perm(lo, hi, 0x5410);
        }
    }
}
// E4M3(x / scale) of V finite values, as IEEE division would have it, mostly without dividing: x times 1 / scale is off by
// less than 2^-22 of itself (two roundings), so the quotient lies between the products with inv (1 - 2^-22) and
// inv (1 + 2^-22); where both round to one code that is the quotient's.  A quotient near the middle between two
// codes, a few of a million, is divided.  (8192 tokens rotated and written: 49.5 us, dividing everything 52.9.)
template <int V> __device__ __forceinline__ void store_codes(uint8_t *p, const float *x, float scale, float inv) {
    constexpr int W = V < 4 ? 1 : V / 4;
    uint32_t w[W], v[W];
    codes_of<V>(w, x, inv * (1.0f - 2.384185791015625e-07f));
    codes_of<V>(v, x, inv * (1.0f + 2.384185791015625e-07f));
    bool same = true;
#pragma unroll
    for (int i = 0; i < W; i++) same = same && w[i] == v[i];
    if (!same) {
        float q[V];
#pragma unroll
        for (int i = 0; i < V; i++) q[i] = x[i] / scale;
        codes_of<V>(w, q, 1.0f);
    }
    if constexpr (V == 1) *p = (uint8_t)w[0];
    else if constexpr (V == 4) *reinterpret_cast<uint32_t *>(p) = w[0];
    else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
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
// PRE rows before anything else; the angles are formed while they are under way.  8192 tokens, 32 + 8 heads of 128, bf16:
// rotated 31 us (5.4 TB/s, 82 % of the measured rate); rotated and written 43.4 (65 %), where 28 M warp instructions take 63 %
// of the issue slots, the cosines' reads, half of them bank conflicts, keep L1's pipe 71 % busy, and 25 warps an SM do not hide both.
template <typename T, int V, int ITER, int PRE, bool HALF>
__global__ void __launch_bounds__(RW_THREADS, ITER == 1 ? 7 : 1) rope_write_kernel(const RopeWrite p) {
    using C = Chunk<T, V>;
    pdl_prologue();
    __shared__ __align__(16) float2 cs_all[RW_TOKENS * 128];
    const int token0 = blockIdx.x * p.tokens_per_cta, n_tokens = min(p.tokens_per_cta, p.tokens - token0);
    const int half = p.rotary / 2;
    const int lpr = p.lanes_per_row, rpc = RW_THREADS / lpr, stride = gridDim.y * rpc;
    const int r = threadIdx.x / lpr, l = threadIdx.x % lpr;
    const int rows = p.nq + p.nk + p.nv, units = p.head_dim / (2 * V), rot_units = half / V;
    bool angles = p.nq + p.nk > 0;
    for (int ti = 0; ti < n_tokens; ti++)
    for (int base = blockIdx.y * rpc; base < rows; base += stride * PRE) {       // the same trips for a whole CTA
        const int token = token0 + ti;
        const float2 *cs = cs_all + ti * 128;
        typename C::Raw raw[PRE][ITER][2];
        size_t off[PRE];                                 // of the row in its tensor
#pragma unroll
        for (int k = 0; k < PRE; k++) {
            const int row = base + k * stride + r;
            const bool is_q = row < p.nq, is_v = row >= p.nq + p.nk;
            const int heads = is_q ? p.nq : is_v ? p.nv : p.nk, head = row - (is_q ? 0 : is_v ? p.nq + p.nk : p.nq);
            off[k] = ((size_t)token * heads + head) * p.head_dim;
            const T *src = (const T *)(is_q ? p.q : is_v ? p.v : p.k) + off[k];
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int u = l + it * lpr;
                if (row >= rows || u >= units) continue;
                const bool halves = HALF && u < rot_units && !is_v;
                const int a = halves ? u * V : u * 2 * V, b = halves ? a + half : a + V;
                raw[k][it][0] = *reinterpret_cast<const typename C::Raw *>(src + a);
                raw[k][it][1] = *reinterpret_cast<const typename C::Raw *>(src + b);
            }
        }
        const uint32_t slot = p.slots ? p.slots[token] : 0u;
        const bool to_cache = p.slots && slot < p.num_slots;
        if (p.slots && !to_cache && slot != 0xFFFFFFFFu && threadIdx.x == 0) report_error(p.err, KERR_SLOT_RANGE);
        if (angles) {                                    // of all the CTA's tokens
            for (int x = threadIdx.x; x < n_tokens * half; x += RW_THREADS) {
                const int at = x / half, i = x - at * half;
                const double turns = (double)p.positions[token0 + at] * (double)p.inv_freq[i] * 0.15915494309189533577;     // 1 / (2 pi)
                float s, co;
                sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
                cs_all[at * 128 + i] = make_float2(co * p.magnitude, s * p.magnitude);
            }
            __syncthreads();
            angles = false;
        }
#pragma unroll
        for (int k = 0; k < PRE; k++) {
            const int row = base + k * stride + r;
            if (base + k * stride >= rows) break;        // the whole CTA
            const bool is_q = row < p.nq, is_v = row >= p.nq + p.nk, quant = is_v || (!is_q && p.k_pool);
            float x[ITER][2 * V];
            int at[ITER], bt[ITER];
            float amax = 0.0f, zero = 0.0f;              // zero: NaN once a value is not finite
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const int u = l + it * lpr;
                const bool on = row < rows && u < units;
                const bool halves = HALF && u < rot_units && !is_v;
                at[it] = !on ? -1 : halves ? u * V : u * 2 * V;
                bt[it] = halves ? at[it] + half : at[it] + V;
                if (!on) continue;
                C::unpack(x[it], raw[k][it][0]);
                C::unpack(x[it] + V, raw[k][it][1]);
                if (!is_v && u * V < half) {
                    if (u * V + V <= half) {
#pragma unroll
                        for (int j = 0; j < V; j++) rotate(x[it][HALF ? j : 2 * j], x[it][HALF ? V + j : 2 * j + 1], cs[u * V + j]);
                    } else if (!HALF) {                  // a unit that the rotated part ends in
#pragma unroll
                        for (int j = 0; j < V; j++)
                            if (u * V + j < half) rotate(x[it][2 * j], x[it][2 * j + 1], cs[u * V + j]);
                    }
                }
                if (quant) {
#pragma unroll
                    for (int j = 0; j < 2 * V; j++) {
                        amax = fmaxf(amax, fabsf(x[it][j]));
                        zero = fmaf(x[it][j], 0.0f, zero);
                    }
                } else {
                    T *out = (T *)(is_q ? p.q_out : p.k_out) + off[k];
                    C::store(out + at[it], x[it]);
                    C::store(out + bt[it], x[it] + V);
                }
            }
            if (!p.slots || !__any_sync(0xffffffffu, quant && row < rows)) continue;
            for (int o = lpr >> 1; o; o >>= 1) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                zero += __shfl_xor_sync(0xffffffffu, zero, o);
            }
            if (!quant || row >= rows || !to_cache) continue;
            const bool finite = zero == 0.0f;
            const float scale = fmaxf(amax / 448.0f, 1.17549435e-38f), inv = 1.0f / scale;
            const int heads = is_v ? p.nv : p.nk, head = row - (is_v ? p.nq + p.nk : p.nq);
            uint8_t *pool = (is_v ? p.v_pool : p.k_pool) + ((size_t)slot * heads + head) * p.head_dim;
            if (l == 0) (is_v ? p.v_scales : p.k_scales)[(size_t)head * p.num_slots + slot] = finite ? scale : __int_as_float(0x7FC00000);
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                if (at[it] < 0) continue;
                if (!finite) {
#pragma unroll
                    for (int j = 0; j < 2 * V; j++) x[it][j] = 0.0f;
                }
                store_codes<V>(pool + at[it], x[it], finite ? scale : 1.0f, finite ? inv : 1.0f);
                store_codes<V>(pool + bt[it], x[it] + V, finite ? scale : 1.0f, finite ? inv : 1.0f);
            }
        }
    }
}

// Rows read back: out[c] = codes of slot indices[c], each head's times its scale; one product and one rounding.  A thread
// takes V codes of one head at a time (32 bytes of output, one store), of N units at once.  HBM-bound: 40001 rows of 1024
// to float32 34.6 us (6.0 TB/s, 91 % of the measured rate; 59.8 with 4 codes a thread).
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
    // Several tokens a CTA, whose threads then all have angles to form, once every SM has CTAs to spare; few tokens are
    // spread over several CTAs each.
    p.tokens = tokens;
    p.tokens_per_cta = tokens >= 16 * sm_count ? RW_TOKENS : tokens >= 8 * sm_count ? 2 : 1;
    const int want = (2 * sm_count + tokens - 1) / tokens;
    const dim3 grid((unsigned)((tokens + p.tokens_per_cta - 1) / p.tokens_per_cta), (unsigned)(want < most ? want : most));
    if (p.split_half)
        return vec ? launch_dependent(rope_write_kernel<T, VEC, 1, 3, true>, grid, dim3(RW_THREADS), 0, s, pdl, p)
                   : launch_dependent(rope_write_kernel<T, 1, 4, 1, true>, grid, dim3(RW_THREADS), 0, s, pdl, p);
    return vec ? launch_dependent(rope_write_kernel<T, VEC, 1, 3, false>, grid, dim3(RW_THREADS), 0, s, pdl, p)
               : launch_dependent(rope_write_kernel<T, 1, 4, 1, false>, grid, dim3(RW_THREADS), 0, s, pdl, p);
}

}  // namespace

cudaError_t launch_rope_write(const RopeWrite &p, int dtype, int tokens, int sm_count, cudaStream_t s, bool pdl) {
    if (tokens <= 0) return cudaSuccess;
    return dtype == DT_BF16 ? rope_write<__nv_bfloat16, 8>(p, tokens, sm_count, s, pdl)
                            : rope_write<float, 4>(p, tokens, sm_count, s, pdl);
}

cudaError_t launch_gather_quant(void *out, int dtype, const uint8_t *pool, const float *scales, const uint32_t *indices,
                                uint32_t kv_dim, uint32_t head_dim, uint32_t num_slots, uint32_t rows, uint32_t *err,
                                int sm_count, cudaStream_t s, bool pdl) {
    if (rows == 0) return cudaSuccess;
    const uint32_t vec = dtype == DT_BF16 ? 16 : 8;      // 32 bytes of output
    const bool ok = head_dim % vec == 0 && (uintptr_t)out % 32 == 0;
    const size_t n = (size_t)(kv_dim / (ok ? vec : 1)) * rows;
    constexpr int N = 4;
    // four units a thread once that still leaves every SM its share of warps; one each below
    const int per = n >= (size_t)4 * 256 * sm_count * 4 ? N : 1;
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
