// Attention over the 8-bit KV cache (E4M3 codes, one float32 scale per slot and KV head; kv_quant.cu).
//
// For query row i (a query token and head), position j visible to it, codes kc_j and vc_j, scales ks_j and vs_j:
//   s_ij = ks_j (q_i . kc_j) / sqrt(head_dim),   o_i = sum_j e^(s_ij - m_i) vs_j vc_j / sum_j e^(s_ij - m_i).
// The scales factor out of both products, so the codes themselves, exact in 16 bits, are what is multiplied.
// Whatever a position that a row does not see holds (codes of an old sequence, a scale that is NaN) is left
// out by selects, never by a weight of zero; rows past kv_len of their request are not read at all.
// A row that sees nothing yields zeros.  Tokens behind the last request are left as they were.
#include <cuda_fp8.h>

#include "kernels.h"
#include "llmrs_common.cuh"
#include "pipeline.cuh"

namespace llmrs {

namespace {

__device__ __forceinline__ float load_f(const void *p, size_t i, int bf16) {
    return bf16 ? bf16_bits_to_f32(((const uint16_t *)p)[i]) : ((const float *)p)[i];
}
__device__ __forceinline__ void store_f(void *p, size_t i, float v, int bf16) {
    if (bf16) ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
    else ((float *)p)[i] = v;
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

// What request `req` brings: its query tokens [first, first + count) and the positions in front of its first
// one.  Lengths that do not fit the page table and starts that do not fit q are cut to what exists.
struct Request {
    int first, count, before;        // query token i sees positions 0 .. before + i
};
__device__ __forceinline__ Request request_of(const AttnQuant &p, int req) {
    const uint32_t a = min(p.query_starts[req], (uint32_t)p.total_q), b = min(p.query_starts[req + 1], (uint32_t)p.total_q);
    const uint32_t room = (uint32_t)min((long long)p.max_blocks * p.block_size, 0x7FFFFFFFll);
    uint32_t len = p.seq_lens[req];
    if (len > room) { report_error(p.err, KERR_SLOT_RANGE); len = room; }
    Request r;
    r.first = (int)a;
    r.count = b > a ? (int)(b - a) : 0;
    r.before = (int)len - r.count;
    return r;
}
// Slot of position `pos`, or -1 (reported) when the page table leads out of the pool.
__device__ __forceinline__ long long slot_of(const AttnQuant &p, int req, int pos) {
    const uint32_t page = p.block_table[(size_t)req * p.max_blocks + pos / p.block_size];
    const unsigned long long slot = (unsigned long long)page * p.block_size + (unsigned)(pos % p.block_size);
    if (slot < p.num_slots) return (long long)slot;
    report_error(p.err, KERR_SLOT_RANGE);
    return -1;
}

// Any head_dim up to 256, F32 or BF16: one CTA per (query token, head).  Thread j forms the score of position
// j of a tile of 128, thread d sums the weighted values of dimension d (and d + 128), with the running maximum
// and sum of a one-pass softmax, all in float32.  Every query head reads its keys and values by itself: this is
// the form for what the tensor-core kernels do not take.
constexpr int AQ_TILE = 128;
__global__ void __launch_bounds__(AQ_TILE) attention_quant_simple_kernel(const AttnQuant p, int bf16) {
    pdl_prologue();
    __shared__ float qs[256], w[AQ_TILE], red[AQ_TILE / 32];
    __shared__ long long slots[AQ_TILE];
    const int head = blockIdx.x % p.n_heads, gq = blockIdx.x / p.n_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int req = 0;
    Request r;
    for (; req < p.num_req; req++) {
        r = request_of(p, req);
        if (gq >= r.first && gq < r.first + r.count) break;
    }
    if (req == p.num_req) return;
    const int len = r.before + gq - r.first + 1;
    const int kvh = head / (p.n_heads / p.n_kv), hd = p.head_dim;
    const size_t q_off = ((size_t)gq * p.n_heads + head) * hd, kv_dim = (size_t)p.n_kv * hd;
    const float *ks = p.k_scales + (size_t)kvh * p.num_slots, *vs = p.v_scales + (size_t)kvh * p.num_slots;
    const float scale = 1.0f / sqrtf((float)hd);
    for (int i = tid; i < hd; i += AQ_TILE) qs[i] = load_f(p.q, q_off + i, bf16) * scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int t0 = 0; t0 < len; t0 += AQ_TILE) {
        const long long slot = t0 + tid < len ? slot_of(p, req, t0 + tid) : -1;
        float s = -INFINITY;
        if (slot >= 0) {
            const uint8_t *k = p.k_pool + (size_t)slot * kv_dim + (size_t)kvh * hd;
            float dot = 0.0f;
            for (int i = 0; i < hd; i++) dot = fmaf(qs[i], e4m3_to_f32(k[i]), dot);
            s = dot * ks[slot];
        }
        bool nan = s != s;                               // fmaxf drops a NaN: carried beside the maximum
        float mx = s;
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) red[warp] = mx;
        slots[tid] = slot;
        nan = __syncthreads_or(nan);
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = nan ? __int_as_float(0x7FC00000) : fmaxf(m, mx);
        const float base = mn == -INFINITY ? 0.0f : mn, f = expf(m - base);
        const float e = slot >= 0 ? expf(s - base) : 0.0f;
        m = mn;
        float sum = e;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        __syncthreads();                                 // the maxima in red[] have been read
        if (lane == 0) red[warp] = sum;
        w[tid] = slot >= 0 ? e * vs[slot] : 0.0f;
        __syncthreads();
        l = l * f + (red[0] + red[1] + red[2] + red[3]);
        const int n = min(AQ_TILE, len - t0);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int d = tid + h * AQ_TILE;
            if (d >= hd) continue;
            float a = acc[h] * f;
            for (int j = 0; j < n; j++)
                if (slots[j] >= 0) a = fmaf(w[j], e4m3_to_f32(p.v_pool[(size_t)slots[j] * kv_dim + (size_t)kvh * hd + d]), a);
            acc[h] = a;
        }
        __syncthreads();                                 // w[], slots[] and red[] are rewritten by the next tile
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int d = tid + h * AQ_TILE;
        if (d < hd) store_f(p.out, q_off + d, l == 0.0f ? 0.0f : acc[h] / l, bf16);
    }
}

}  // namespace

cudaError_t launch_attention_quant(const AttnQuant &p, int dtype, cudaStream_t s, bool pdl, uint64_t *launches) {
    if (p.total_q <= 0 || p.num_req <= 0) return cudaSuccess;
    ++*launches;
    return launch_dependent(attention_quant_simple_kernel, dim3((unsigned)p.total_q * p.n_heads), dim3(AQ_TILE), 0, s, pdl, p,
                            (int)(dtype == DT_BF16));
}

}  // namespace llmrs
