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
__device__ __forceinline__ float4 load4(const void *p, size_t i, int bf16) {
    if (!bf16) return *reinterpret_cast<const float4 *>((const float *)p + i);
    const uint2 u = *reinterpret_cast<const uint2 *>((const uint16_t *)p + i);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ void store4(void *p, size_t i, float4 v, int bf16) {
    if (bf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2 *>((__nv_bfloat16 *)p + i) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        *reinterpret_cast<float4 *>((float *)p + i) = v;
    }
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

constexpr int SHORT_ROWS = 16;       // a request of at most this many rows (query tokens x group) is a short one

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

// ---- few rows: requests that decode ---------------------------------------------------------------
// HBM-bound: a position's 2 head_dim codes and two scales are read once for all the query rows of its KV head.
//
// Work.  A row block is up to RB rows (query token x head of the group) of one request and KV head; a unit is a
// row block's next 16 PW positions, PW = 8 / HW, for HW KV heads at once.  The units of all requests form one
// sequence that is cut into equal contiguous ranges, one per CTA, so ragged batches load every SM alike and one
// long request spreads over the whole GPU.  The lengths are on the device, so each CTA adds them up itself.  A row
// block that lies in several ranges leaves (accumulator, maximum, sum) in the workspace for the merge kernel.
//
// A CTA has 8 warps, HW heads x PW runs of 16 positions, so that neighbouring heads of a slot, neighbours in memory,
// are read at the same time.  Each warp is on its own: it fetches its 16 positions NST units ahead into its own
// ring by 16-byte asynchronous copies, and meets other warps only at the end of a row block.
//
// Arithmetic (mma m16n8k16, f16 operands, float32 sums): E4M3 codes are exact in f16; bf16 queries are too, once a row is
// scaled by a power of two.  TERMS = 2 (F32) splits queries and weights into a high and a low f16.  The order in which
// dimensions enter a dot product is free as long as both operands agree, so a lane takes 16 consecutive codes of a
// row as its part of four products; codes of values come transposed by ldmatrix in pairs of dimensions, which one
// byte permute turns into pairs of positions.  A weight enters as w = e^(s - m) vs / R * 2^15 with R the least power of two
// that no vs so far exceeds: f16 keeps it to 2^-11 (bf16: 2^-8), and down to 2^-40 of the largest.
constexpr int SH_WARPS = 8, SH_THREADS = 32 * SH_WARPS;
constexpr int SH_MIN_UNITS = 4;      // a CTA gets at least this many units: shorter ranges cost more in merging than they save

template <int HD> struct ShortStage {
    static constexpr int K = 0, V = 16 * HD, KS = 32 * HD, VS = KS + 64, MASK = VS + 64, BYTES = MASK + 16;
};

struct Rows {                        // what both kernels need to know about the split into rows and units
    int rb, tp, hw, only_short;      // rows per block, positions per unit, KV heads per CTA, leave requests of more than SHORT_ROWS rows out
};
__device__ __forceinline__ void shape_of(const AttnQuant &p, const Rows &w, const Request &r, int &blocks, int &tiles) {
    const long long rows = (long long)r.count * (p.n_heads / p.n_kv);
    blocks = w.only_short && rows > SHORT_ROWS ? 0 : (int)((rows + w.rb - 1) / w.rb);
    const int len = r.before + r.count;
    tiles = len > 0 ? (int)(((long long)len + w.tp - 1) / w.tp) : 1;     // a row block that sees nothing still writes its zeros
}
// All threads of the CTA: the units of all requests (returned), and into found[] the request that holds unit
// `want(total)` and the units before that request; or, with `req` >= 0, the units before that request.
template <typename Want>
__device__ __forceinline__ long long scan_units(const AttnQuant &p, const Rows &w, long long *sums, long long *found, Want want, int req) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    auto units = [&](int r) -> long long {
        if (r >= p.num_req) return 0;
        int b, t;
        shape_of(p, w, request_of(p, r), b, t);
        return (long long)b * t;
    };
    const long long mine = units(tid);                   // the first blockDim.x requests stay in registers
    long long s = mine;
    for (int r = tid + blockDim.x; r < p.num_req; r += blockDim.x) s += units(r);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    long long total = 0;
    for (int i = 0; i < warps; i++) total += sums[i];
    __syncthreads();
    const long long at = want(total);
    long long base = 0;
    for (int r0 = 0; r0 < p.num_req; r0 += blockDim.x) {
        const long long u = r0 == 0 ? mine : units(r0 + tid);
        long long inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        long long before = base + inc - u;
        for (int i = 0; i < warp; i++) before += sums[i];
        if (req >= 0 ? r0 + tid == req : (u > 0 && at >= before && at < before + u)) { found[0] = r0 + tid; found[1] = before; }
        for (int i = 0; i < warps; i++) base += sums[i];
        __syncthreads();
    }
    return total;
}
// CTAs (per head group) that share `total` units, and the range of one; the CTA that holds unit u.
__device__ __forceinline__ int sharers(long long total, int ctas) {
    const long long most = (total + SH_MIN_UNITS - 1) / SH_MIN_UNITS;
    return (int)min((long long)ctas, max(most, 1ll));
}
__device__ __forceinline__ long long first_unit(long long total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int holder(long long total, int n, long long u) { return (int)(((u + 1) * n - 1) / total); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two E4M3 codes (low, high byte) -> f16x2, exact.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// What the f16 pair lost of (lo, hi), as an f16 pair.
__device__ __forceinline__ uint32_t pack_f16_rest(float lo, float hi, uint32_t kept) {
    const __half2 k = *reinterpret_cast<const __half2 *>(&kept);
    return pack_f16(lo - __low2float(k), hi - __high2float(k));
}
__device__ __forceinline__ void copy16_or_zero(void *dst, const void *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_or_zero(void *dst, const void *src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void *row) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(row)));
}
// The power of two by which a row of queries with largest magnitude `amax` enters as f16 (its largest then in
// [2^13, 2^14)): 2^e, |e| <= 126.  Rows of zeros and rows that are not finite stay as they are.
__device__ __forceinline__ int row_exponent(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);    // biased; amax >= 0
    return amax == 0.0f || e == 255 ? 0 : max(-126, min(126, 13 - (e - 127)));
}

template <int HD, int RB, int TERMS, int HW, int NST>
__global__ void __launch_bounds__(SH_THREADS, RB == 8 && TERMS == 1 ? 2 : 1)
attention_quant_short_kernel(const AttnQuant p, int bf16, int only_short, float *__restrict__ ws) {
    pdl_prologue();
    using St = ShortStage<HD>;
    constexpr int PW = SH_WARPS / HW, TP = 16 * PW, KS = HD / 16, CH = HD / 16;
    constexpr int HALVES = RB / 8;                       // 8 rows: the lower half of the 16-row operand stays zero
    extern __shared__ __align__(128) uint8_t sh_smem[];
    __shared__ long long sums[SH_WARPS], found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int groups = p.n_kv / HW, hg = blockIdx.x % groups, cta = blockIdx.x / groups, ctas = gridDim.x / groups;
    const int kvh = hg * HW + warp / PW, wp = warp % PW;
    const int group = p.n_heads / p.n_kv;
    const Rows rows{RB, TP, HW, only_short};
    found[0] = -1;
    int n_cta = 1;
    const long long total = scan_units(p, rows, sums, found, [&](long long all) {
        n_cta = sharers(all, ctas);
        return cta < n_cta ? first_unit(all, n_cta, cta) : -1ll;
    }, -1);
    if (cta >= n_cta || total == 0) return;
    const long long u_begin = first_unit(total, n_cta, cta), u_end = first_unit(total, n_cta, cta + 1);
    int req = (int)found[0];
    long long req_base = found[1];                       // units before request `req`

    uint8_t *ring = sh_smem + (size_t)warp * NST * St::BYTES;
    const size_t kv_dim = (size_t)p.n_kv * HD;
    const uint8_t *kp = p.k_pool + (size_t)kvh * HD, *vp = p.v_pool + (size_t)kvh * HD;
    const float *ksp = p.k_scales + (size_t)kvh * p.num_slots, *vsp = p.v_scales + (size_t)kvh * p.num_slots;

    for (long long u = u_begin; u < u_end;) {
        int blocks, tiles;
        const Request r = request_of(p, req);
        shape_of(p, rows, r, blocks, tiles);
        if (u >= req_base + (long long)blocks * tiles) { req_base += (long long)blocks * tiles; req++; continue; }
        const int rb = (int)((u - req_base) / tiles), t0 = (int)((u - req_base) % tiles);
        const int t1 = (int)min((long long)tiles, t0 + (u_end - u));
        // ---- the rows of this block: rows g and g + 8 are this lane's ----
        const int n_rows = min(RB, r.count * group - rb * RB);
        const int kv_end = r.before + (rb * RB + n_rows - 1) / group + 1;
        int len[2];
        size_t q_off[2];
        uint32_t qa[TERMS][KS][4];
        float c_row[2];                                  // what turns a product of codes into a score in units of log2
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = g + 8 * h, rr = rb * RB + i;
            const bool on = h < HALVES && i < n_rows;
            len[h] = on ? r.before + rr / group + 1 : 0;
            q_off[h] = on ? ((size_t)(r.first + rr / group) * p.n_heads + (size_t)kvh * group + rr % group) * HD : 0;
            c_row[h] = 0.0f;
#pragma unroll
            for (int x = 0; x < TERMS; x++)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) qa[x][ks][h] = qa[x][ks][2 + h] = 0u;
            if (h >= HALVES) continue;
            // the lane's dimensions: 16 (t + 4 hf) + 4 w + (0 .. 3) of step 4 hf + w
            float amax = 0.0f;
            float q[KS][4];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float4 v = on ? load4(p.q, q_off[h] + 16 * (t + 4 * (ks / 4)) + 4 * (ks % 4), bf16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                q[ks][0] = v.x; q[ks][1] = v.y; q[ks][2] = v.z; q[ks][3] = v.w;
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = row_exponent(amax);
            const float up = exp2i(ex);
            c_row[h] = exp2i(-ex) * (1.4426950408889634f / sqrtf((float)HD));
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float a = q[ks][2 * e] * up, b = q[ks][2 * e + 1] * up;
                    qa[0][ks][h + 2 * e] = pack_f16(a, b);
                    if (TERMS == 2) qa[TERMS - 1][ks][h + 2 * e] = pack_f16_rest(a, b, qa[0][ks][h + 2 * e]);
                }
        }
        float o[CH][2][4];                               // [chunk of 16 dims][even, odd dims][row g: 4t + par, 4t + 2 + par; row g + 8]
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int x = 0; x < 2; x++) o[c][x][0] = o[c][x][1] = o[c][x][2] = o[c][x][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        uint32_t r_bits = 17u << 23;                     // R: a power of two, at least 2^-110

        const int n_steps = min(t1, (max(kv_end, 0) + TP - 1) / TP) - t0;        // at most 0: nothing to see in this range
        const int j = lane & 15;
        auto page_of = [&](int i) -> uint32_t {          // page table entry of this lane's position of step i
            const int pos = (t0 + i) * TP + wp * 16 + j;
            return i < n_steps && pos < kv_end ? p.block_table[(size_t)req * p.max_blocks + pos / p.block_size] : 0u;
        };
        uint32_t page = page_of(0);
        auto fetch = [&](int i) {
            if (i < n_steps) {
                uint8_t *st = ring + (i % NST) * St::BYTES;
                const int pos = (t0 + i) * TP + wp * 16 + j;
                const unsigned long long s64 = (unsigned long long)page * p.block_size + (unsigned)(pos % p.block_size);
                const bool ok = pos < kv_end && s64 < p.num_slots;
                if (pos < kv_end && !ok) report_error(p.err, KERR_SLOT_RANGE);
                const uint32_t slot = ok ? (uint32_t)s64 : 0u;
                const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xFFFFu;
                if (lane == 0) *reinterpret_cast<uint32_t *>(st + St::MASK) = mask;
                copy4_or_zero(st + (lane < 16 ? St::KS : St::VS) + 4 * j, (lane < 16 ? ksp : vsp) + slot, ok);
                constexpr int RPI = 32 / CH;             // rows per pass of the warp
                const int c = lane % CH;
#pragma unroll
                for (int k = 0; k < 16 / RPI; k++) {
                    const int row = lane / CH + RPI * k;
                    const size_t off = (size_t)__shfl_sync(0xffffffffu, slot, row) * kv_dim + 16 * c;
                    const bool on = mask >> row & 1;
                    // chunks of a row are permuted so that fragment reads fall on distinct banks
                    copy16_or_zero(st + St::K + row * HD + 16 * (c ^ (HD == 128 ? (row & 1) << 2 : 0)), kp + off, on);
                    copy16_or_zero(st + St::V + row * HD + 16 * (c ^ (HD == 128 ? row & 7 : (row >> 1) & 3)), vp + off, on);
                }
                page = page_of(i + 1);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < NST - 1; i++) fetch(i);
        for (int i = 0; i < n_steps; i++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
            __syncwarp();                                // this step's bytes are there for all lanes, the last step's are no longer read
            fetch(i + NST - 1);
            const uint8_t *st = ring + (i % NST) * St::BYTES;
            // ---- scores of the warp's 16 positions: two groups of eight ----
            float s[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
                const int row = 8 * nt + g;
#pragma unroll
                for (int hf = 0; hf < KS / 4; hf++) {
                    const int c = HD == 128 ? (t + 4 * hf) ^ ((row & 1) << 2) : t;
                    const uint4 w4 = *reinterpret_cast<const uint4 *>(st + St::K + row * HD + 16 * c);
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const uint32_t b0 = codes_to_f16(w[x] & 0xFFFFu), b1 = codes_to_f16(w[x] >> 16);
#pragma unroll
                        for (int y = 0; y < TERMS; y++) mma_f16(s[nt], qa[y][4 * hf + x], b0, b1);
                    }
                }
            }
            const uint32_t mask = *reinterpret_cast<const uint32_t *>(st + St::MASK);
            const float *ks = reinterpret_cast<const float *>(st + St::KS), *vs = reinterpret_cast<const float *>(st + St::VS);
            float vw[2][2], vmax = 0.0f;
            const int p0 = (t0 + i) * TP + wp * 16;
            float mx[2] = {-INFINITY, -INFINITY};
            bool seen[2][2][2];                          // [half][group][element]
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
                const float2 k2 = *reinterpret_cast<const float2 *>(ks + 8 * nt + 2 * t), v2 = *reinterpret_cast<const float2 *>(vs + 8 * nt + 2 * t);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int at = 8 * nt + 2 * t + e;
                    const bool ok = mask >> at & 1;
                    vw[nt][e] = e ? v2.y : v2.x;
                    vmax = fmaxf(vmax, vw[nt][e]);
#pragma unroll
                    for (int h = 0; h < HALVES; h++) {
                        seen[h][nt][e] = ok && p0 + at < len[h];
                        const float x = s[nt][2 * h + e] * ((e ? k2.y : k2.x) * c_row[h]);
                        s[nt][2 * h + e] = seen[h][nt][e] ? x : -INFINITY;
                        mx[h] = fmaxf(mx[h], s[nt][2 * h + e]);
                    }
                }
            }
            vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
            vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
            const uint32_t r_new = max(r_bits, min((__float_as_uint(vmax) + 0x7FFFFFu) & 0x7F800000u, 253u << 23));
            const float shrink = __uint_as_float(r_bits - r_new + (127u << 23));         // R / R', zero when that is below 2^-126
            float f[2];
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float mn = fmaxf(m[h], mx[h]);
                mx[h] = mn == -INFINITY ? 0.0f : mn;     // a row that has seen nothing yet
                f[h] = mn == m[h] ? 1.0f : ex2(m[h] - mx[h]);
                m[h] = mn;
            }
            const bool moved = r_new != r_bits || f[0] != 1.0f || (HALVES == 2 && f[HALVES - 1] != 1.0f);
            if (__any_sync(0xffffffffu, moved)) {
                const float sh = r_new - r_bits >= (127u << 23) ? 0.0f : shrink;
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            o[c][x][2 * h] *= f[h] * sh;
                            o[c][x][2 * h + 1] *= f[h] * sh;
                        }
#pragma unroll
                for (int h = 0; h < HALVES; h++) l[h] *= f[h];
                r_bits = r_new;
            }
            const float inv_r = __uint_as_float(((127u + 127u + 15u) << 23) - r_bits);   // 2^15 / R
            uint32_t pa[TERMS][4];
#pragma unroll
            for (int x = 0; x < TERMS; x++) pa[x][1] = pa[x][3] = 0u;
#pragma unroll
            for (int nt = 0; nt < 2; nt++)
#pragma unroll
                for (int h = 0; h < HALVES; h++) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float x = ex2(s[nt][2 * h + e] - mx[h]);
                        l[h] += x;
                        w[e] = seen[h][nt][e] ? x * (vw[nt][e] * inv_r) : 0.0f;
                    }
                    pa[0][h + 2 * nt] = pack_f16(w[0], w[1]);
                    if (TERMS == 2) pa[TERMS - 1][h + 2 * nt] = pack_f16_rest(w[0], w[1], pa[0][h + 2 * nt]);
                }
            // ---- weighted values ----
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                // matrices (positions 0-7, chunk c), (8-15, c), (0-7, c + 1), (8-15, c + 1)
                const int row = (lane & 7) + 8 * (lane >> 3 & 1), ch = c + (lane >> 4);
                uint32_t b[4];
                ldmatrix_x4_trans(b, st + St::V + row * HD + 16 * (ch ^ (HD == 128 ? row & 7 : (row >> 1) & 3)));
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t lo = __byte_perm(b[2 * x], 0, 0x3120), hi = __byte_perm(b[2 * x + 1], 0, 0x3120);
#pragma unroll
                    for (int par = 0; par < 2; par++) {
                        const uint32_t b0 = codes_to_f16(par ? lo >> 16 : lo & 0xFFFFu), b1 = codes_to_f16(par ? hi >> 16 : hi & 0xFFFFu);
#pragma unroll
                        for (int y = 0; y < TERMS; y++) mma_f16(o[c + x][par], pa[y], b0, b1);
                    }
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();                                    // the ring may be filled again
        // ---- the row block's part is done: out, or into the workspace ----
        const float back = __uint_as_float(r_bits - (15u << 23));        // R / 2^15
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = blockIdx.x * 2 + (u == u_begin ? 0 : 1);
        float *ws_o = ws + (size_t)slot * HW * RB * HD;
        float2 *ws_ml = reinterpret_cast<float2 *>(ws + (size_t)gridDim.x * 2 * HW * RB * HD) + (size_t)slot * HW * RB;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        if constexpr (PW == 1) {
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                const int i = g + 8 * h;
                if (i >= n_rows) continue;
                const float norm = whole ? (l[h] == 0.0f ? 0.0f : back / l[h]) : back;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    const float4 v = make_float4(o[c][0][2 * h] * norm, o[c][1][2 * h] * norm, o[c][0][2 * h + 1] * norm, o[c][1][2 * h + 1] * norm);
                    const int d = 16 * c + 4 * t;
                    if (whole) store4(p.out, q_off[h] + d, v, bf16);
                    else *reinterpret_cast<float4 *>(ws_o + ((size_t)(warp / PW) * RB + i) * HD + d) = v;
                }
                if (!whole && t == 0) ws_ml[(warp / PW) * RB + i] = make_float2(m[h], l[h]);
            }
        } else {
            // the PW warps of a head meet in shared memory: [warp][row][HD] and [warp][row] {maximum, sum}
            float *po = reinterpret_cast<float *>(sh_smem);
            float2 *pml = reinterpret_cast<float2 *>(po + SH_WARPS * RB * HD);
            __syncthreads();                             // every warp has left its ring
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                const int i = g + 8 * h;
#pragma unroll
                for (int c = 0; c < CH; c++)
                    *reinterpret_cast<float4 *>(po + ((size_t)warp * RB + i) * HD + 16 * c + 4 * t) =
                        make_float4(o[c][0][2 * h] * back, o[c][1][2 * h] * back, o[c][0][2 * h + 1] * back, o[c][1][2 * h + 1] * back);
                if (t == 0) pml[warp * RB + i] = make_float2(m[h], l[h]);
            }
            __syncthreads();
            for (int x = tid; x < HW * n_rows * (HD / 4); x += SH_THREADS) {
                const int d = 4 * (x % (HD / 4)), i = x / (HD / 4) % n_rows, hd = x / (HD / 4) / n_rows;
                float mm = -INFINITY;
#pragma unroll
                for (int w = 0; w < PW; w++) mm = fmaxf(mm, pml[(hd * PW + w) * RB + i].x);
                const float base = mm == -INFINITY ? 0.0f : mm;
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float ll = 0.0f;
#pragma unroll
                for (int w = 0; w < PW; w++) {
                    const float2 ml = pml[(hd * PW + w) * RB + i];
                    const float wt = ex2(ml.x - base);
                    const float4 v = *reinterpret_cast<const float4 *>(po + ((size_t)(hd * PW + w) * RB + i) * HD + d);
                    ll = fmaf(ml.y, wt, ll);
                    a.x = fmaf(v.x, wt, a.x); a.y = fmaf(v.y, wt, a.y); a.z = fmaf(v.z, wt, a.z); a.w = fmaf(v.w, wt, a.w);
                }
                if (whole) {
                    const float norm = ll == 0.0f ? 0.0f : 1.0f / ll;
                    const int rr = rb * RB + i;
                    const size_t off = ((size_t)(r.first + rr / group) * p.n_heads + (size_t)(hg * HW + hd) * group + rr % group) * HD + d;
                    store4(p.out, off, make_float4(a.x * norm, a.y * norm, a.z * norm, a.w * norm), bf16);
                } else {
                    *reinterpret_cast<float4 *>(ws_o + ((size_t)hd * RB + i) * HD + d) = a;
                    if (d == 0) ws_ml[hd * RB + i] = make_float2(mm, ll);
                }
            }
            __syncthreads();                             // the ring may be filled again
        }
        u += t1 - t0;
    }
}

// One CTA per (query token, head): the parts of its row, if they were left by several CTAs, joined in order.  A
// quarter (head_dim 64: an eighth) of a warp's lanes would do for a part; HD / 4 threads take one each round.
constexpr int MERGE_THREADS = 512;
template <int HD>
__global__ void __launch_bounds__(MERGE_THREADS)
attention_quant_merge_kernel(const AttnQuant p, int bf16, const Rows rows, int ctas, const float *__restrict__ ws) {
    pdl_prologue();
    constexpr int PER = MERGE_THREADS / (HD / 4);        // parts at a time
    __shared__ long long sums[MERGE_THREADS / 32], found[2];
    __shared__ float4 acc_s[MERGE_THREADS];
    __shared__ float red[MERGE_THREADS / 32], lsum[PER];
    const int head = blockIdx.x % p.n_heads, gq = blockIdx.x / p.n_heads, tid = threadIdx.x;
    const int group = p.n_heads / p.n_kv, kvh = head / group;
    int req = 0;
    Request r;
    for (; req < p.num_req; req++) {
        r = request_of(p, req);
        if (gq >= r.first && gq < r.first + r.count) break;
    }
    if (req == p.num_req) return;
    const long long total = scan_units(p, rows, sums, found, [](long long) { return 0ll; }, req);
    int blocks, tiles;
    shape_of(p, rows, r, blocks, tiles);
    if (blocks == 0) return;                             // the other kernel's
    const int rr = (gq - r.first) * group + head % group, rb = rr / rows.rb, i = rr % rows.rb;
    const int n = sharers(total, ctas), groups = p.n_kv / rows.hw, hg = kvh / rows.hw, hd = kvh % rows.hw;
    const long long a = found[1] + (long long)rb * tiles;
    const int c0 = holder(total, n, a), c1 = holder(total, n, a + tiles - 1);
    if (c0 == c1) return;                                // one CTA had all of it and wrote the row
    const size_t slots = (size_t)ctas * groups * 2;
    const float2 *ml = reinterpret_cast<const float2 *>(ws + slots * rows.hw * rows.rb * HD);
    auto part = [&](int c) {                             // index of CTA c's part of this row
        const int which = max(a, first_unit(total, n, c)) == first_unit(total, n, c) ? 0 : 1;
        return ((size_t)((c * groups + hg) * 2 + which) * rows.hw + hd) * rows.rb + i;
    };
    float m = -INFINITY;
    for (int c = c0 + tid; c <= c1; c += MERGE_THREADS) m = fmaxf(m, ml[part(c)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < MERGE_THREADS / 32; w++) m = fmaxf(m, red[w]);
    const float base = m == -INFINITY ? 0.0f : m;
    const int d = 4 * (tid % (HD / 4)), lane_part = tid / (HD / 4);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int c = c0 + lane_part; c <= c1; c += PER) {
        const size_t x = part(c);
        const float2 v = ml[x];
        const float4 q = *reinterpret_cast<const float4 *>(ws + x * HD + d);
        const float w = ex2(v.x - base);
        l = fmaf(v.y, w, l);
        acc.x = fmaf(q.x, w, acc.x); acc.y = fmaf(q.y, w, acc.y); acc.z = fmaf(q.z, w, acc.z); acc.w = fmaf(q.w, w, acc.w);
    }
    acc_s[tid] = acc;
    if (d == 0) lsum[lane_part] = l;
    __syncthreads();
    if (tid >= HD / 4) return;
    float ll = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int x = 0; x < PER; x++) {
        const float4 q = acc_s[x * (HD / 4) + tid];
        ll += lsum[x];
        acc.x += q.x; acc.y += q.y; acc.z += q.z; acc.w += q.w;
    }
    const float norm = ll == 0.0f ? 0.0f : 1.0f / ll;
    store4(p.out, ((size_t)gq * p.n_heads + head) * HD + d, make_float4(acc.x * norm, acc.y * norm, acc.z * norm, acc.w * norm), bf16);
}

struct ShortPlan { int rb, terms, hw, stages, per_sm; };
ShortPlan short_plan(const AttnQuant &p, int dtype) {
    const int group = p.n_heads / p.n_kv;
    ShortPlan s;
    s.rb = group <= 8 && p.total_q <= p.num_req ? 8 : 16;
    s.terms = dtype == DT_F32 ? 2 : 1;
    s.hw = p.n_kv % 8 == 0 ? 8 : p.n_kv % 4 == 0 ? 4 : p.n_kv % 2 == 0 ? 2 : 1;
    s.per_sm = s.rb == 8 && s.terms == 1 ? 2 : 1;
    s.stages = s.per_sm == 2 ? 3 : 6;
    return s;
}
int short_grid(const AttnQuant &p, const ShortPlan &s, int sm_count) {
    const int groups = p.n_kv / s.hw, per = s.per_sm * sm_count / groups;
    return (per < 1 ? 1 : per) * groups;
}
size_t short_workspace(const AttnQuant &p, const ShortPlan &s, int sm_count) {
    return (size_t)short_grid(p, s, sm_count) * 2 * s.hw * s.rb * (p.head_dim + 2) * sizeof(float);
}

template <int HD, int RB, int TERMS, int HW, int NST>
cudaError_t launch_short(const AttnQuant &p, int dtype, int grid, int only_short, float *ws, cudaStream_t s, bool pdl) {
    constexpr size_t ring = (size_t)SH_WARPS * NST * ShortStage<HD>::BYTES;
    constexpr size_t meet = HW == SH_WARPS ? 0 : (size_t)SH_WARPS * RB * (HD + 2) * sizeof(float);
    constexpr size_t smem = ring > meet ? ring : meet;
    auto k = attention_quant_short_kernel<HD, RB, TERMS, HW, NST>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(k, dim3((unsigned)grid), dim3(SH_THREADS), smem, s, pdl, p, (int)(dtype == DT_BF16), only_short, ws);
}
template <int HD, int RB, int TERMS, int NST>
cudaError_t launch_short_hw(const AttnQuant &p, int dtype, int hw, int grid, int only_short, float *ws, cudaStream_t s, bool pdl) {
    switch (hw) {
        case 8: return launch_short<HD, RB, TERMS, 8, NST>(p, dtype, grid, only_short, ws, s, pdl);
        case 4: return launch_short<HD, RB, TERMS, 4, NST>(p, dtype, grid, only_short, ws, s, pdl);
        case 2: return launch_short<HD, RB, TERMS, 2, NST>(p, dtype, grid, only_short, ws, s, pdl);
        default: return launch_short<HD, RB, TERMS, 1, NST>(p, dtype, grid, only_short, ws, s, pdl);
    }
}
template <int HD>
cudaError_t launch_short_all(const AttnQuant &p, int dtype, const ShortPlan &pl, int sm_count, int only_short, float *ws, cudaStream_t s, bool pdl) {
    const int grid = short_grid(p, pl, sm_count);
    cudaError_t e;
    if (pl.terms == 2) e = pl.rb == 8 ? launch_short_hw<HD, 8, 2, 6>(p, dtype, pl.hw, grid, only_short, ws, s, pdl)
                                      : launch_short_hw<HD, 16, 2, 6>(p, dtype, pl.hw, grid, only_short, ws, s, pdl);
    else e = pl.rb == 8 ? launch_short_hw<HD, 8, 1, 3>(p, dtype, pl.hw, grid, only_short, ws, s, pdl)
                        : launch_short_hw<HD, 16, 1, 6>(p, dtype, pl.hw, grid, only_short, ws, s, pdl);
    if (e != cudaSuccess) return e;
    const Rows rows{pl.rb, 16 * SH_WARPS / pl.hw, pl.hw, only_short};
    return launch_dependent(attention_quant_merge_kernel<HD>, dim3((unsigned)p.total_q * p.n_heads), dim3(MERGE_THREADS), 0, s, pdl,
                            p, (int)(dtype == DT_BF16), rows, grid / (p.n_kv / pl.hw), (const float *)ws);
}

bool mma_supported(const AttnQuant &p) { return p.head_dim == 64 || p.head_dim == 128; }

}  // namespace

size_t attention_quant_workspace(const AttnQuant &p, int dtype, int sm_count) {
    return mma_supported(p) ? short_workspace(p, short_plan(p, dtype), sm_count) : 0;
}

cudaError_t launch_attention_quant(const AttnQuant &p, int dtype, float *ws, int sm_count, cudaStream_t s, bool pdl,
                                   uint64_t *launches) {
    if (p.total_q <= 0 || p.num_req <= 0) return cudaSuccess;
    if (!mma_supported(p)) {
        ++*launches;
        return launch_dependent(attention_quant_simple_kernel, dim3((unsigned)p.total_q * p.n_heads), dim3(AQ_TILE), 0, s, pdl, p,
                                (int)(dtype == DT_BF16));
    }
    const ShortPlan pl = short_plan(p, dtype);
    *launches += 2;
    return p.head_dim == 128 ? launch_short_all<128>(p, dtype, pl, sm_count, 0, ws, s, pdl)
                             : launch_short_all<64>(p, dtype, pl, sm_count, 0, ws, s, pdl);
}

}  // namespace llmrs
