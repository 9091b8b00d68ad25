// Attention over the 8-bit KV cache (E4M3 codes, one float32 scale per slot and KV head; kv_quant.cu).
//
// For query row i (a query token and head), position j visible to it, codes kc_j and vc_j, scales ks_j and vs_j:
//   s_ij = ks_j (q_i . kc_j) / sqrt(head_dim),   o_i = sum_j e^(s_ij - m_i) vs_j vc_j / sum_j e^(s_ij - m_i).
// The scales factor out of both products, so the codes themselves, exact in 16 bits, are what is multiplied.
// Whatever a position that a row does not see holds (codes of an old sequence, a scale that is NaN) is left
// out by selects, never by a weight of zero; rows past kv_len of their request are not read at all.
// A row that sees nothing yields zeros.  Tokens behind the last request are left as they were.
#include <cuda_fp8.h>

#include <type_traits>

#include "kernels.h"
#include "llmrs_common.cuh"
#include "pipeline.cuh"
#include "tensor_map.h"
#include "umma.cuh"

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
__device__ __forceinline__ void store2(void *p, size_t i, float2 v, int bf16) {
    if (bf16) *reinterpret_cast<__nv_bfloat162 *>((__nv_bfloat16 *)p + i) = __floats2bfloat162_rn(v.x, v.y);
    else *reinterpret_cast<float2 *>((float *)p + i) = v;
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
    const uint32_t room = (uint32_t)min((long long)p.max_blocks * p.block_size, 0x7FFF0000ll);      // positions, rounded up to tiles, stay ints
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
// row block's next 32 PW positions, PW = 4 / HW, for HW KV heads at once.  The units of all requests form one
// sequence that is cut into equal contiguous ranges, one per CTA, so ragged batches load every SM alike and one
// long request spreads over the whole GPU.  The lengths are on the device, so each CTA adds them up itself.  A row
// block that lies in several ranges leaves (accumulator, maximum, sum) parts in the workspace; the last CTA to finish of
// each 18 neighbours joins theirs, and the last of those the rest, always in the order of the parts (few requests:
// attention_quant_merge_kernel).
//
// One request of 131071 positions: 56 us, 76 % of the measured HBM rate; without the joining 48 (88 %).  64 requests of
// 100 to 8192: 108 us, 79 %; without 97 (88 %).
//
// A CTA has 4 consumer warps, HW heads x PW times 32 positions, so that neighbouring heads of a slot, neighbours
// in memory, are read at the same time (one head a CTA: 142 us for the 64 requests; 16 positions a warp instead of 32: 69 us
// instead of 60 for the one, at that step), and a producer that keeps NST units in flight, through to the end of the
// CTA's range.  Where 16 positions never straddle a page (block_size a multiple of 16, and the scales' rows 16-byte
// aligned) the producer is one thread that issues four tiled TMA copies per 16 positions of all the heads; otherwise
// four warps fetch 16 bytes a lane.  (The first form had every warp fetch for itself: 692 instructions a warp per 16
// positions, and one request of 131071 positions took 88 us, bound by issue slots at 48 % of HBM.)
//
// Arithmetic (mma m16n8k16, f16 operands, float32 sums): E4M3 codes are exact in f16; bf16 queries are too, once a row is
// scaled by a power of two.  TERMS = 2 (F32) splits queries and weights into a high and a low f16.  Positions (for the
// second product: dimensions) are the 16 rows of an operand and query rows the 8 columns, so 8 rows need one
// product for what would take two the other way round; the weights change sides by movmatrix.  The order in
// which dimensions enter a dot product is free as long as both operands agree, so a lane takes 16 consecutive codes
// of a row as its part of four products; codes of values come transposed by ldmatrix in pairs of dimensions, which
// one byte permute turns into pairs of positions.
//
// A weight enters as w = e^s vs / 2^a * 2^15, where a is the row's own: at least the largest s + log2 vs among the positions
// that it has seen, and at most 10 more, so f16 keeps a weight to 2^-11 (bf16: 2^-8), and down to 2^-30 of the largest, whatever
// other rows see and however large a value of little weight is.  Where the vs of the 32 positions
// of a step lie within 2^10 of one another, the largest s of the row plus log2 of the largest vs does for a, and one exponential
// does for the weight and the sum; elsewhere a is found position by position, and a weight has an exponential of its own.
constexpr int SH_WARPS = 4, SH_THREADS = 32 * SH_WARPS;      // consumers
constexpr int SH_GR = 2;             // runs of 16 positions that a warp takes at a time
constexpr int SH_TILES = SH_WARPS * SH_GR;                   // (run, head) tiles of a unit
constexpr int SH_MIN_UNITS = 4;      // a CTA gets at least this many units: shorter ranges cost more in merging than they save

template <int HD, int HW> struct ShortStage {
    static constexpr int RUNS = SH_TILES / HW, TILE = SH_TILES * 16 * HD, BYTES = 2 * TILE;   // codes: keys, then values
    // scales (RUN bytes for 16 positions of HW heads; a TMA copy starts on 128 bytes) and which positions are there
    static constexpr int RUN = HW == 1 ? 128 : 64 * HW, KS = 0, VS = RUNS * RUN, MASK = 2 * VS, AUX = MASK + 128;
};
struct ShortMaps { CUtensorMap k, v, ks, vs; };

struct Rows {                        // what both kernels need to know about the split into rows and units
    int rb, tp, hw, only_short;      // rows per block, positions per unit, KV heads per CTA, leave requests of more than SHORT_ROWS rows out
};
__device__ __forceinline__ void shape_of(const AttnQuant &p, const Rows &w, const Request &r, int &blocks, int &tiles) {
    const long long rows = (long long)r.count * (p.n_heads / p.n_kv);
    blocks = w.only_short && rows > SHORT_ROWS ? 0 : (int)((rows + w.rb - 1) / w.rb);
    const int len = r.before + r.count;
    tiles = len > 0 ? (int)(((long long)len + w.tp - 1) / w.tp) : 1;     // a row block that sees nothing still writes its zeros
}
// A whole warp, every warp for itself: the units of all requests (returned), and the request that holds unit
// want(total), its data and the units before it.
struct Found {
    int req;
    Request r;
    long long before;
};
template <typename Want>
__device__ __forceinline__ long long scan_units(const AttnQuant &p, const Rows &w, Want want, Found &found) {
    const int lane = threadIdx.x & 31;
    auto units = [&](int req, Request &r) -> long long {
        if (req >= p.num_req) return 0;
        int b, t;
        r = request_of(p, req);
        shape_of(p, w, r, b, t);
        return (long long)b * t;
    };
    Request r0 = {0, 0, 0};
    const long long u0 = units(lane, r0);                // the first 32 requests stay in registers
    long long total = u0;
#pragma unroll 4
    for (int q = lane + 32; q < p.num_req; q += 32) {
        Request r;
        total += units(q, r);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const long long at = want(total);
    if (at < 0 || total == 0) return total;
    long long base = 0;
    for (int q0 = 0; q0 < p.num_req; q0 += 32) {
        Request r = r0;
        const long long u = q0 == 0 ? u0 : units(q0 + lane, r);
        long long inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, at < base + inc);       // the first of them holds it: empty ones have inc as before
        if (hit) {
            const int src = __ffs(hit) - 1;
            found.req = q0 + src;
            found.r.first = __shfl_sync(0xffffffffu, r.first, src);
            found.r.count = __shfl_sync(0xffffffffu, r.count, src);
            found.r.before = __shfl_sync(0xffffffffu, r.before, src);
            found.before = base + __shfl_sync(0xffffffffu, inc - u, src);
            return total;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    return total;
}
constexpr int SH_JOIN = 18;          // parts that are joined at once: two levels reach two CTAs on each of 148 SMs
// CTAs (per head group) that share `total` units, and the range of one; the CTA that holds unit u.
__device__ __forceinline__ int sharers(long long total, int ctas) {
    const long long most = (total + SH_MIN_UNITS - 1) / SH_MIN_UNITS;
    return (int)min((long long)min(ctas, SH_JOIN * (SH_JOIN - 1)), max(most, 1ll));      // what two levels of joining reach
}
__device__ __forceinline__ long long first_unit(long long total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int holder(long long total, int n, long long u) { return (int)(((u + 1) * n - 1) / total); }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four E4M3 codes -> two f16x2 (low bytes first), exact.
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
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
// Arrives on `bar` (one of its expected arrivals) once this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const void *tmap, int c0, int c1, int c2, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void *row) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(row)));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {             // of an 8x8 matrix of 16-bit values
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// The power of two by which a row of queries with largest magnitude `amax` enters as f16 (its largest then in
// [2^13, 2^14)): 2^e, |e| <= 126.  Rows of zeros and rows that are not finite stay as they are.
__device__ __forceinline__ int row_exponent(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);    // biased; amax >= 0
    return amax == 0.0f || e == 255 ? 0 : max(-126, min(126, 13 - (e - 127)));
}
// Powers of two, as a float's bits: the one at or below a size, the least that it does not exceed; between 2^-126 and 2^126.
__device__ __forceinline__ uint32_t power_of(float size) { return max(1u << 23, min(__float_as_uint(size) & 0x7F800000u, 253u << 23)); }
__device__ __forceinline__ uint32_t power_above(float size) { return max(1u << 23, min((__float_as_uint(size) + 0x7FFFFFu) & 0x7F800000u, 253u << 23)); }
__device__ __forceinline__ float log2_of(uint32_t power_bits) { return (float)((int)(power_bits >> 23) - 127); }
// 16-byte chunk c of row `row` of a tile of HD-byte rows, as the 128- and 64-byte swizzles of TMA place it.
template <int HD> __device__ __forceinline__ int chunk_at(int row, int c) {
    return row * HD + 16 * (c ^ (HD == 128 ? row & 7 : (row >> 1) & 3));
}

// A CTA's way through its range of units: one row block (or the part of it in the range) after the other.
struct Segment {
    Request r;
    int req, rb, t0, t1, tiles, n_rows, kv_end, n_steps;
    long long item;                  // the row block's first unit
    bool first;                      // starts where the range starts
};
template <int RB, int TP> struct Walk {
    long long u, u_begin, u_end, req_base;
    int req;
    Request r;                       // of `req`
    __device__ __forceinline__ bool next(const AttnQuant &p, const Rows &w, Segment &s) {
        while (u < u_end) {
            int blocks;
            shape_of(p, w, r, blocks, s.tiles);
            if (u >= req_base + (long long)blocks * s.tiles) {
                req_base += (long long)blocks * s.tiles;
                r = request_of(p, ++req);
                continue;
            }
            s.r = r;
            const int group = p.n_heads / p.n_kv;
            s.req = req;
            s.rb = (int)((u - req_base) / s.tiles);
            s.t0 = (int)((u - req_base) % s.tiles);
            s.t1 = (int)min((long long)s.tiles, s.t0 + (u_end - u));
            s.n_rows = min(RB, s.r.count * group - s.rb * RB);
            s.kv_end = s.r.before + (s.rb * RB + s.n_rows - 1) / group + 1;
            s.n_steps = max(0, min(s.t1, (max(s.kv_end, 0) + TP - 1) / TP) - s.t0);   // 0: nothing to see in this range
            s.first = u == u_begin;
            s.item = u - s.t0;
            u += s.t1 - s.t0;
            return true;
        }
        return false;
    }
};

// Loads that stay where they are, in front of what uses them, and come from L2 (other CTAs have just written there).
__device__ __forceinline__ float4 load_part4(const float *p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float2 load_part2(const float2 *p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
// The consumer warps of a CTA.  bar.sync is .aligned: lanes that left a loop or a branch before the others meet them first.
__device__ __forceinline__ void consumers_sync() {
    __syncwarp();
    named_barrier_sync(1, SH_THREADS);
}
struct Join {
    void *out;
    float *ws;
    float2 *ws_ml;
    int bf16, n_heads, group, first_head;                // of the HW KV heads
    int first_token, first_row, n_rows;                  // the request's first query token, the row block's first row
    int n, slot0, step, slot1;                           // part 0 is in slot slot0, part i > 0 in slot1 + (i - 1) * step
    bool last;
};
// The consumer threads of a CTA: joins n parts of HW heads x n_rows rows, into the output (`last`) or into the first of
// their slots.  Four elements (16 bytes) of the result a thread and two parts of each at a time, with their maxima and
// sums: 16 loads under way (four parts at a time: 112 us instead of 108 for 64 ragged requests).
template <int HD, int RB, int HW>
__device__ __noinline__ void join_parts(const Join &j) {     // not inlined: its registers are not the main loop's
    constexpr int E = 4, B = 2;
    const int tid = threadIdx.x, n = j.n, n_rows = j.n_rows, rows = HW * n_rows, elems = rows * (HD / 4);
    const int inv_rows = 65536 / n_rows + 1;             // r / n_rows = r * inv_rows >> 16 for r < 64, n_rows <= 16
    float *ws = j.ws;
    float2 *ws_ml = j.ws_ml;
    for (int x0 = tid; x0 - tid < elems; x0 += E * SH_THREADS) {
        int row[E], d[E];
        float m[E], l[E];
        float4 a[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int x = min(x0 + e * SH_THREADS, elems - 1), r = x / (HD / 4);        // past the end: the last one again, not stored
            const int head = r * inv_rows >> 16;
            row[e] = head * RB + r - head * n_rows;
            d[e] = 4 * (x % (HD / 4));
            m[e] = -INFINITY;
            l[e] = 0.0f;
            a[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (int y0 = 0; y0 < n; y0 += B) {
            float4 v[B][E];
            float2 ml[B][E];
#pragma unroll
            for (int y = 0; y < B; y++) {
                const int i = min(y0 + y, n - 1);
                const size_t slot = (size_t)(i ? j.slot1 + (i - 1) * j.step : j.slot0) * HW * RB;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    ml[y][e] = load_part2(ws_ml + slot + row[e]);
                    v[y][e] = load_part4(ws + (slot + row[e]) * HD + d[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                float mn = m[e];
#pragma unroll
                for (int y = 0; y < B; y++) mn = fmaxf(mn, ml[y][e].x);
                const float base = mn == -INFINITY ? 0.0f : mn, f = ex2(m[e] - base);
                m[e] = mn;
                l[e] *= f;
                a[e].x *= f; a[e].y *= f; a[e].z *= f; a[e].w *= f;
#pragma unroll
                for (int y = 0; y < B; y++) {
                    if (y0 + y >= n) break;
                    const float w = ex2(ml[y][e].x - base);
                    l[e] = fmaf(ml[y][e].y, w, l[e]);
                    a[e].x = fmaf(v[y][e].x, w, a[e].x); a[e].y = fmaf(v[y][e].y, w, a[e].y);
                    a[e].z = fmaf(v[y][e].z, w, a[e].z); a[e].w = fmaf(v[y][e].w, w, a[e].w);
                }
            }
        }
        if (!j.last) consumers_sync();    // every thread has read the maxima and sums of slot `to` for its row
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int x = x0 + e * SH_THREADS;
            if (x >= elems) break;
            if (j.last) {
                const float norm = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
                const int rr = j.first_row + row[e] % RB;
                store4(j.out, ((size_t)(j.first_token + rr / j.group) * j.n_heads + (size_t)(j.first_head + row[e] / RB) * j.group + rr % j.group) * HD + d[e],
                       make_float4(a[e].x * norm, a[e].y * norm, a[e].z * norm, a[e].w * norm), j.bf16);
            } else {                                     // this thread alone has read the element that it overwrites
                const size_t at = (size_t)j.slot0 * HW * RB + row[e];
                *reinterpret_cast<float4 *>(ws + at * HD + d[e]) = a[e];
                if (d[e] == 0) ws_ml[at] = make_float2(m[e], l[e]);
            }
        }
    }
}
// Counts this CTA in; true in the one that completes `n`, which also clears the counter for the next launch.  The barrier
// orders the CTA's writes before the count, whose release makes them visible to whoever counts later and acquires.
__device__ __forceinline__ bool last_of(uint32_t *counter, uint32_t n, uint32_t *flag) {
    consumers_sync();
    if (threadIdx.x == 0) {
        uint32_t before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
        if (before == n - 1) *counter = 0;
        *flag = before == n - 1;
    }
    consumers_sync();
    return *flag != 0;
}

template <int HD, int RB, int TERMS, int HW, int NST, bool TMA>
__global__ void __launch_bounds__(SH_THREADS + (TMA ? 32 : 128), 2)
attention_quant_short_kernel(const __grid_constant__ ShortMaps maps, const AttnQuant p, int bf16, int only_short, uint32_t polls,
                             float *__restrict__ ws, uint32_t *__restrict__ counters, int join_here) {
    using St = ShortStage<HD, HW>;
    constexpr int PW = SH_WARPS / HW, RUNS = St::RUNS, TP = 16 * RUNS, KS = HD / 16, CH = HD / 16, NT = RB / 8;
    constexpr int PASS = 1;                              // chunks of 16 dimensions the warps of a head exchange at a time
    extern __shared__ __align__(1024) uint8_t sh_smem[];
    uint8_t *codes = sh_smem, *aux = codes + NST * St::BYTES;
    float *meet = reinterpret_cast<float *>(aux + NST * St::AUX);            // PW > 1: [warp][row][16 PASS] and [warp][row] {max, sum}
    __shared__ uint32_t is_last;
    __shared__ __align__(8) uint64_t full[NST], empty[NST];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < NST; i++) {
            mbar_init(&full[i], TMA ? 1 : 128 + 4);
            mbar_init(&empty[i], SH_WARPS);
        }
        mbar_init_fence();
    }
    __syncthreads();
    pdl_prologue();
    const int groups = p.n_kv / HW, hg = blockIdx.x % groups, cta = blockIdx.x / groups, ctas = gridDim.x / groups;
    const int group = p.n_heads / p.n_kv;
    const Rows rows{RB, TP, HW, only_short};
    int n_cta = 1;
    Found found;
    const long long total = scan_units(p, rows, [&](long long all) {
        n_cta = sharers(all, ctas);
        return cta < n_cta ? first_unit(all, n_cta, cta) : -1ll;
    }, found);
    if (cta >= n_cta || total == 0) return;              // the same for every warp
    Walk<RB, TP> walk;
    walk.u = walk.u_begin = first_unit(total, n_cta, cta);
    walk.u_end = first_unit(total, n_cta, cta + 1);
    walk.req = found.req;
    walk.req_base = found.before;
    walk.r = found.r;
    Segment s;
    int stage = 0;
    uint32_t phase = 0;
    bool dead = false;                                   // a wait was given up: go on without waiting, so that no barrier is missed

    if (warp >= SH_WARPS) {
        // ---- producer ----
        int issued = 0;
        auto given = [&]() {                             // is the stage free?  All lanes go on or none does
            dead = !__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, polls));
            if (dead && lane == 0) report_error(p.err, KERR_EMPTY_WAIT);
            return !dead;
        };
        while (!dead && walk.next(p, rows, s)) {
            const uint32_t *table = p.block_table + (size_t)s.req * p.max_blocks;
            if constexpr (TMA) {
                // lane x looks up run `r0 + x` of the segment (16 positions each, RUNS to a step); the copies then go out in order
                for (int r0 = 0; r0 < s.n_steps * RUNS && !dead; r0 += 32) {
                    const int pos = s.t0 * TP + 16 * (r0 + lane);
                    int slot = (int)p.num_slots, n_ok = 0;               // out of range: zeros, nothing read
                    if (r0 + lane < s.n_steps * RUNS && pos < s.kv_end) {
                        const unsigned long long s64 = (unsigned long long)table[pos / p.block_size] * p.block_size + (unsigned)(pos % p.block_size);
                        const int want = min(16, s.kv_end - pos);
                        if (s64 < p.num_slots) { slot = (int)s64; n_ok = (int)min((unsigned long long)want, p.num_slots - s64); }
                        if (n_ok < want) report_error(p.err, KERR_SLOT_RANGE);
                    }
                    const int steps = min(32 / RUNS, s.n_steps - r0 / RUNS);
                    for (int i = 0; i < steps && !dead; i++) {
                        if (issued >= NST && !given()) break;
                        uint8_t *cd = codes + stage * St::BYTES, *ax = aux + stage * St::AUX;
                        if (lane / RUNS == i) reinterpret_cast<uint32_t *>(ax + St::MASK)[lane % RUNS] = (1u << n_ok) - 1;
                        __syncwarp();
                        if (lane == 0) mbar_arrive_expect_tx(&full[stage], St::BYTES + 2 * SH_TILES * 64);
                        __syncwarp();
#pragma unroll
                        for (int x = 0; x < RUNS; x++) {
                            const int at = __shfl_sync(0xffffffffu, slot, i * RUNS + x);
                            if (lane == 0) {
                                tma_load_3d(cd + x * HW * 16 * HD, &maps.k, 0, at, hg * HW, &full[stage]);
                                tma_load_3d(cd + St::TILE + x * HW * 16 * HD, &maps.v, 0, at, hg * HW, &full[stage]);
                                tma_load_2d(ax + St::KS + x * St::RUN, &maps.ks, at, hg * HW, &full[stage]);
                                tma_load_2d(ax + St::VS + x * St::RUN, &maps.vs, at, hg * HW, &full[stage]);
                            }
                        }
                        issued++;
                        if (++stage == NST) { stage = 0; phase ^= 1; }
                    }
                }
            } else {
                // four warps, two of the eight tiles of 16 positions each
                const size_t kv_dim = (size_t)p.n_kv * HD;
                const int pw = warp - SH_WARPS, j = lane & 15;
                auto page_of = [&](int i, int run) -> uint32_t {
                    const int pos = (s.t0 + i) * TP + run * 16 + j;
                    return i < s.n_steps && pos < s.kv_end ? table[pos / p.block_size] : 0u;
                };
                uint32_t page[2] = {page_of(0, 2 * pw / HW), page_of(0, (2 * pw + 1) / HW)};
                for (int i = 0; i < s.n_steps; i++) {
                    if (issued >= NST && !given()) break;
                    uint8_t *cd = codes + stage * St::BYTES, *ax = aux + stage * St::AUX;
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const int sub = 2 * pw + y, run = sub / HW, head = hg * HW + sub % HW;
                        const int pos = (s.t0 + i) * TP + run * 16 + j;
                        const unsigned long long s64 = (unsigned long long)page[y] * p.block_size + (unsigned)(pos % p.block_size);
                        const bool ok = pos < s.kv_end && s64 < p.num_slots;
                        if (pos < s.kv_end && !ok) report_error(p.err, KERR_SLOT_RANGE);
                        const uint32_t slot = ok ? (uint32_t)s64 : 0u;
                        const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xFFFFu;
                        if (lane == 0) reinterpret_cast<uint32_t *>(ax + St::MASK)[sub] = mask;
                        copy4_or_zero(ax + (lane < 16 ? St::KS : St::VS) + run * St::RUN + sub % HW * 64 + 4 * j,
                                      (lane < 16 ? p.k_scales : p.v_scales) + (size_t)head * p.num_slots + slot, ok);
                        constexpr int RPI = 32 / CH;     // rows per pass of the warp
                        const int c = lane % CH;
#pragma unroll
                        for (int k = 0; k < 16 / RPI; k++) {
                            const int row = lane / CH + RPI * k;
                            const size_t off = (size_t)__shfl_sync(0xffffffffu, slot, row) * kv_dim + (size_t)head * HD + 16 * c;
                            const bool on = mask >> row & 1;
                            copy16_or_zero(cd + sub * 16 * HD + chunk_at<HD>(row, c), p.k_pool + off, on);
                            copy16_or_zero(cd + St::TILE + sub * 16 * HD + chunk_at<HD>(row, c), p.v_pool + off, on);
                        }
                        page[y] = page_of(i + 1, run);
                    }
                    copies_arrive(&full[stage]);
                    if (lane == 0) mbar_arrive(&full[stage]);            // the masks
                    issued++;
                    if (++stage == NST) { stage = 0; phase ^= 1; }
                }
            }
        }
        // no copy may be in flight when the CTA ends: the last ones issued have landed once their barriers have turned
        for (int i = 0; i < min(issued, NST); i++) {
            if (stage-- == 0) { stage = NST - 1; phase ^= 1; }
            mbar_wait(&full[stage], phase, polls);
        }
        return;
    }

    // ---- consumers ----
    constexpr int GR = SH_GR;
    const int hw = warp % HW, wp = warp / HW, kvh = hg * HW + hw, first_tile = wp * GR * HW + hw;
    while (walk.next(p, rows, s)) {
        // rows: this lane loads the queries of row g (and g + 8) as operand columns; scores and sums come out for rows 2t, 2t + 1 (+ 8)
        uint32_t qb[TERMS][NT][KS][2];
        float c_row[NT][2];                              // what turns a product of codes into a score in units of log2
        int len[NT][2];
        const int min_len = s.r.before + s.rb * RB / group + 1;          // what the first row sees
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int i = g + 8 * n, rr = s.rb * RB + i;
            const bool on = i < s.n_rows;
            const size_t off = on ? ((size_t)(s.r.first + rr / group) * p.n_heads + (size_t)kvh * group + rr % group) * HD : 0;
            float q[KS][4], amax = 0.0f;
            // the lane's dimensions: 16 (t + 4 hf) + 4 w + (0 .. 3) of step 4 hf + w
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float4 v = on ? load4(p.q, off + 16 * (t + 4 * (ks / 4)) + 4 * (ks % 4), bf16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                q[ks][0] = v.x; q[ks][1] = v.y; q[ks][2] = v.z; q[ks][3] = v.w;
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = row_exponent(amax);
            const float up = exp2i(ex), c = exp2i(-ex) * (1.4426950408889634f / sqrtf((float)HD));
            const int visible = on ? s.r.before + rr / group + 1 : 0;
#pragma unroll
            for (int e = 0; e < 2; e++) {                // row 2t + e is lane 4 (2t + e)'s
                c_row[n][e] = __shfl_sync(0xffffffffu, c, 4 * (2 * t + e));
                len[n][e] = __shfl_sync(0xffffffffu, visible, 4 * (2 * t + e));
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float a = q[ks][2 * e] * up, b = q[ks][2 * e + 1] * up;
                    qb[0][n][ks][e] = pack_f16(a, b);
                    if (TERMS == 2) qb[TERMS - 1][n][ks][e] = pack_f16_rest(a, b, qb[0][n][ks][e]);
                }
        }
        // [rows 8n ..][chunk of 16 dims]: dims 16c + 2g (0, 1) and 16c + 2g + 1 (2, 3) of rows 2t (0, 2) and 2t + 1 (1, 3)
        float o[NT][CH][4];
        float m[NT][2], l[NT][2], a[NT][2];              // O counts in 2^(a - 15)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = a[n][0] = a[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.0f;
        }
        for (int i = 0; i < s.n_steps; i++) {
            if (!dead && !mbar_wait(&full[stage], phase, polls)) { dead = true; report_error(p.err, KERR_FULL_WAIT); }
            __syncwarp();                                // what follows is .aligned
            uint8_t *kt = codes + stage * St::BYTES + first_tile * 16 * HD, *vt = kt + St::TILE;
            const uint8_t *ax = aux + stage * St::AUX;
            const int p0 = (s.t0 + i) * TP + wp * 16 * GR;
            uint32_t mask[GR];
            float kw[GR][2], vw[GR][2];                  // scales of positions g and g + 8 of each run
            bool all = p0 + 16 * GR <= min_len;          // every row sees every position
#pragma unroll
            for (int r = 0; r < GR; r++) {
                mask[r] = reinterpret_cast<const uint32_t *>(ax + St::MASK)[TMA ? wp * GR + r : first_tile + r * HW];
                all = all && mask[r] == 0xFFFFu;
                const float *ks = reinterpret_cast<const float *>(ax + (wp * GR + r) * St::RUN) + 16 * hw, *vs = ks + St::VS / 4;
                kw[r][0] = ks[g]; kw[r][1] = ks[g + 8];
                vw[r][0] = vs[g]; vw[r][1] = vs[g + 8];
            }
            // ---- scores: positions g and g + 8 of each run against rows 2t, 2t + 1 ----
            float sc[GR][NT][4];
#pragma unroll
            for (int r = 0; r < GR; r++) {
#pragma unroll
                for (int n = 0; n < NT; n++) sc[r][n][0] = sc[r][n][1] = sc[r][n][2] = sc[r][n][3] = 0.0f;
#pragma unroll
                for (int hf = 0; hf < KS / 4; hf++) {
                    const uint4 wa = *reinterpret_cast<const uint4 *>(kt + r * HW * 16 * HD + chunk_at<HD>(g, t + 4 * hf));
                    const uint4 wb = *reinterpret_cast<const uint4 *>(kt + r * HW * 16 * HD + chunk_at<HD>(g + 8, t + 4 * hf));
                    const uint32_t w0[4] = {wa.x, wa.y, wa.z, wa.w}, w1[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        uint32_t a[4];
                        codes_to_f16(w0[x], a[0], a[2]);
                        codes_to_f16(w1[x], a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int y = 0; y < TERMS; y++) mma_f16(sc[r][n], a, qb[y][n][4 * hf + x][0], qb[y][n][4 * hf + x][1]);
                    }
                }
            }
            // ---- what a row does not see, the running maxima, the sizes of what is summed, the weights ----
#pragma unroll
            for (int r = 0; r < GR; r++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = 0; x < 4; x++) sc[r][n][x] *= kw[r][x >> 1] * c_row[n][x & 1];
            if (!all) {
#pragma unroll
                for (int r = 0; r < GR; r++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const bool ok = mask[r] >> (g + 8 * h) & 1;
                        if (!ok) vw[r][h] = 0.0f;
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (!ok || p0 + 16 * r + g + 8 * h >= len[n][e]) sc[r][n][2 * h + e] = -INFINITY;
                    }
                    if (TMA && mask[r] != 0xFFFFu) {     // rows of no position: their weight is zero, but their bytes may be NaN codes
                        uint8_t *v = vt + r * HW * 16 * HD;
                        for (int row = __popc(mask[r]) + lane / CH; row < 16; row += 32 / CH)
                            *reinterpret_cast<uint4 *>(v + row * HD + 16 * (lane % CH)) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before a copy writes there again
                    }
                }
                __syncwarp();
            }
            float vmax = 0.0f, av[GR][2];                // sizes of the values' scales (0: not finite)
#pragma unroll
            for (int r = 0; r < GR; r++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    av[r][h] = fabsf(vw[r][h]) <= 3.402823466e38f ? fabsf(vw[r][h]) : 0.0f;
                    vmax = fmaxf(vmax, av[r][h]);
                }
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, x));
            const uint32_t v_bits = power_above(vmax);
            const float v_log = log2_of(v_bits);
            bool near = true;                            // those that are there are of sizes within 2^10 of one another
#pragma unroll
            for (int r = 0; r < GR; r++)
#pragma unroll
                for (int h = 0; h < 2; h++) near = near && (av[r][h] >= __uint_as_float(v_bits) * 0x1p-10f || !(mask[r] >> (g + 8 * h) & 1));
            float mn[NT][2], an[NT][2], top[NT][2], ref[NT][2];          // the new m and a; m and what scores count from, finite
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = fmaxf(sc[0][n][e], sc[0][n][2 + e]);
#pragma unroll
                    for (int r = 1; r < GR; r++) mx = fmaxf(mx, fmaxf(sc[r][n][e], sc[r][n][2 + e]));
#pragma unroll
                    for (int x = 4; x <= 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                    mn[n][e] = fmaxf(m[n][e], mx);
                    an[n][e] = fmaxf(a[n][e], mx + v_log);               // at least the largest s + log2 vs that the row sees
                    top[n][e] = mn[n][e] == -INFINITY ? 0.0f : mn[n][e]; // a row that has seen nothing yet
                    ref[n][e] = (an[n][e] == -INFINITY ? 0.0f : an[n][e]) - (15.0f + v_log);
                    near = near && ref[n][e] - top[n][e] <= 80.0f;       // the sum keeps its weights above float32's least
                }
            near = __all_sync(0xffffffffu, near);
            if (!near) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float mv = -INFINITY;
#pragma unroll
                        for (int r = 0; r < GR; r++)
#pragma unroll
                            for (int h = 0; h < 2; h++)
                                if (av[r][h] > 0.0f) mv = fmaxf(mv, sc[r][n][2 * h + e] + log2_of(power_above(av[r][h])));
#pragma unroll
                        for (int x = 4; x <= 16; x <<= 1) mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, x));
                        an[n][e] = fmaxf(a[n][e], mv);
                        ref[n][e] = an[n][e] == -INFINITY ? 0.0f : an[n][e];
                    }
            }
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) moved = moved || mn[n][e] != m[n][e] || an[n][e] != a[n][e];
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (mn[n][e] != m[n][e]) l[n][e] *= ex2(m[n][e] - mn[n][e]);
                        const float f = an[n][e] == a[n][e] ? 1.0f : ex2(a[n][e] - an[n][e]);
#pragma unroll
                        for (int c = 0; c < CH; c++) { o[n][c][e] *= f; o[n][c][2 + e] *= f; }
                        m[n][e] = mn[n][e];
                        a[n][e] = an[n][e];
                    }
            }
            uint32_t pb[TERMS][GR][NT][2];
            auto weights = [&](auto near_tag) {
                constexpr bool NEAR = decltype(near_tag)::value;
                float sum[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++) sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
                for (int r = 0; r < GR; r++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t by = NEAR ? v_bits : power_of(av[r][h]);  // a value by itself: vs = 2^own times its rest
                        const float vr = vw[r][h] * __uint_as_float((254u << 23) - by), own = 15.0f + log2_of(by);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float w[2];
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                // (scores and references, large numbers that are alike, are subtracted before anything else: that is exact)
                                const float score = sc[r][n][2 * h + e], x = ex2(score - (NEAR ? ref[n][e] : top[n][e]));
                                sum[n][e] += x;
                                w[e] = NEAR ? x * vr : score == -INFINITY ? 0.0f : ex2((score - ref[n][e]) + own) * vr;      // not 0 * NaN
                            }
                            const uint32_t hi = pack_f16(w[0], w[1]);
                            pb[0][r][n][h] = transposed(hi);
                            if (TERMS == 2) pb[TERMS - 1][r][n][h] = transposed(pack_f16_rest(w[0], w[1], hi));
                        }
                    }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) l[n][e] += NEAR ? sum[n][e] * ex2(ref[n][e] - top[n][e]) : sum[n][e];
            };
            if (near) weights(std::true_type{});
            else weights(std::false_type{});
            // ---- weighted values: 16 dimensions a product ----
#pragma unroll
            for (int r = 0; r < GR; r++)
#pragma unroll
                for (int c = 0; c < CH; c += 2) {
                    // matrices (positions 0-7, chunk c), (8-15, c), (0-7, c + 1), (8-15, c + 1)
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, vt + r * HW * 16 * HD + chunk_at<HD>((lane & 7) + 8 * (lane >> 3 & 1), c + (lane >> 4)));
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        uint32_t a[4];
                        codes_to_f16(__byte_perm(b[2 * x], 0, 0x3120), a[0], a[1]);
                        codes_to_f16(__byte_perm(b[2 * x + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int y = 0; y < TERMS; y++) mma_f16(o[n][c + x], a, pb[y][r][n][0], pb[y][r][n][1]);
                    }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
            if (++stage == NST) { stage = 0; phase ^= 1; }
        }
        // ---- the row block's part is done: out, or into the workspace ----
        float back[NT][2][2];                            // 2^(a - 15 - m), in two factors: each stays in float32's range
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x = a[n][e] == -INFINITY ? -INFINITY : (a[n][e] - m[n][e]) - 15.0f, y = truncf(0.5f * x);
                back[n][e][0] = x == -INFINITY ? 0.0f : ex2(y);
                back[n][e][1] = x == -INFINITY ? 0.0f : ex2(x - y);
            }
        const bool whole = s.t0 == 0 && s.t1 == s.tiles;
        const int slot = blockIdx.x * 2 + (s.first ? 0 : 1);
        float *ws_o = ws + (size_t)slot * HW * RB * HD;
        float2 *ws_ml = reinterpret_cast<float2 *>(ws + (size_t)gridDim.x * 2 * HW * RB * HD) + (size_t)slot * HW * RB;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
        if constexpr (PW == 1) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = 8 * n + 2 * t + e, rr = s.rb * RB + i;
                    if (i >= s.n_rows) continue;
                    const float b0 = back[n][e][0], b1 = whole ? (l[n][e] == 0.0f ? 0.0f : back[n][e][1] / l[n][e]) : back[n][e][1];
                    const size_t off = ((size_t)(s.r.first + rr / group) * p.n_heads + (size_t)kvh * group + rr % group) * HD;
#pragma unroll
                    for (int c = 0; c < CH; c++) {
                        const float2 v = make_float2(o[n][c][e] * b0 * b1, o[n][c][2 + e] * b0 * b1);
                        if (whole) store2(p.out, off + 16 * c + 2 * g, v, bf16);
                        else *reinterpret_cast<float2 *>(ws_o + ((size_t)hw * RB + i) * HD + 16 * c + 2 * g) = v;
                    }
                    if (!whole && g == 0) ws_ml[hw * RB + i] = make_float2(m[n][e], l[n][e]);
                }
        } else {
            // the PW warps of a head meet in shared memory, 16 PASS dimensions at a time
            constexpr int D = 16 * PASS;
            float2 *ml = reinterpret_cast<float2 *>(meet + SH_WARPS * RB * D);
#pragma unroll
            for (int c0 = 0; c0 < CH; c0 += PASS) {
                consumers_sync();       // what was there has been read
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int i = 8 * n + 2 * t + e;
#pragma unroll
                        for (int c = 0; c < PASS; c++)
                            *reinterpret_cast<float2 *>(meet + ((size_t)warp * RB + i) * D + 16 * c + 2 * g) =
                                make_float2(o[n][c0 + c][e] * back[n][e][0] * back[n][e][1], o[n][c0 + c][2 + e] * back[n][e][0] * back[n][e][1]);
                        if (g == 0) ml[warp * RB + i] = make_float2(m[n][e], l[n][e]);
                    }
                consumers_sync();
                for (int x = tid; x < HW * s.n_rows * (D / 4); x += SH_THREADS) {
                    const int d = 4 * (x % (D / 4)), i = x / (D / 4) % s.n_rows, hd = x / (D / 4) / s.n_rows;
                    float mm = -INFINITY;
#pragma unroll
                    for (int w = 0; w < PW; w++) mm = fmaxf(mm, ml[(w * HW + hd) * RB + i].x);
                    const float base = mm == -INFINITY ? 0.0f : mm;
                    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float ll = 0.0f;
#pragma unroll
                    for (int w = 0; w < PW; w++) {
                        const float2 v2 = ml[(w * HW + hd) * RB + i];
                        const float wt = ex2(v2.x - base);
                        const float4 v = *reinterpret_cast<const float4 *>(meet + ((size_t)(w * HW + hd) * RB + i) * D + d);
                        ll = fmaf(v2.y, wt, ll);
                        a.x = fmaf(v.x, wt, a.x); a.y = fmaf(v.y, wt, a.y); a.z = fmaf(v.z, wt, a.z); a.w = fmaf(v.w, wt, a.w);
                    }
                    if (whole) {
                        const float norm = ll == 0.0f ? 0.0f : 1.0f / ll;
                        const int rr = s.rb * RB + i;
                        const size_t off = ((size_t)(s.r.first + rr / group) * p.n_heads + (size_t)(hg * HW + hd) * group + rr % group) * HD;
                        store4(p.out, off + 16 * c0 + d, make_float4(a.x * norm, a.y * norm, a.z * norm, a.w * norm), bf16);
                    } else {
                        *reinterpret_cast<float4 *>(ws_o + ((size_t)hd * RB + i) * HD + 16 * c0 + d) = a;
                        if (c0 == 0 && d == 0) ws_ml[hd * RB + i] = make_float2(mm, ll);
                    }
                }
            }
        }
        if (whole || !join_here) continue;
        const int c0 = holder(total, n_cta, s.item), c1 = holder(total, n_cta, s.item + s.tiles - 1);
        const int g0 = cta / SH_JOIN * SH_JOIN, gf = max(c0, g0), gl = min(c1, g0 + SH_JOIN - 1);    // of these neighbours
        // a CTA's first part, or its second if the row block starts within its range, which only the first holder's can
        const int inside = s.item > first_unit(total, n_cta, c0) ? 1 : 0;
        auto slot_of_cta = [&](int c) { return (c * groups + hg) * 2 + (c == c0 ? inside : 0); };
        const bool near = gf == c0 && gl == c1;
        Join j;
        j.out = p.out; j.ws = ws; j.ws_ml = reinterpret_cast<float2 *>(ws + (size_t)gridDim.x * 2 * HW * RB * HD);
        j.bf16 = bf16; j.n_heads = p.n_heads; j.group = group; j.first_head = hg * HW;
        j.first_token = s.r.first; j.first_row = s.rb * RB; j.n_rows = s.n_rows;
        j.n = gl - gf + 1; j.slot0 = slot_of_cta(gf); j.slot1 = slot_of_cta(gf + 1); j.step = 2 * groups;
        j.last = near;
        if (!last_of(counters + j.slot0, (uint32_t)j.n, &is_last)) continue;
        join_parts<HD, RB, HW>(j);
        if (near) continue;
        j.n = c1 / SH_JOIN - c0 / SH_JOIN + 1; j.slot0 = slot_of_cta(c0); j.slot1 = slot_of_cta((c0 / SH_JOIN + 1) * SH_JOIN);
        j.step = 2 * groups * SH_JOIN;
        j.last = true;
        if (last_of(counters + gridDim.x * 2 + j.slot0, (uint32_t)j.n, &is_last)) join_parts<HD, RB, HW>(j);
    }
}

// ---- many rows: prompts and chunks of prompts -------------------------------------------------------
// The floor is the tensor cores' (tcgen05, f16 operands, float32 accumulators in TMEM), then the exponentials': a score costs
// 4 head_dim operations, 512 of a tensor core's cycles for 128 x 128 of them, and one ex2, 1024 cycles of the
// SM's 16 a cycle.  So a CTA keeps two tiles of 128 query rows (token x head of the group, packed) against one
// stream of keys and values: while one tile's weights are formed the tensor cores work for the other.
//
//   warps 0-3, 4-7   weights of tile 0, 1: a thread owns a row.  Scores come from TMEM 16 columns at a time, weights go back
//                    as f16 over the scores that they came from.
//   warps 8-11, 12-15   keys, values: codes to shared memory as they are, one tile ahead, then to f16 in the 128-byte
//                    swizzle; the scales beside them.  Any page size: rows are looked up one by one.
//   warp 16          issues the products: S = Q K^T (both from shared memory), O += W V (W from TMEM; the values lie
//                    as they come, positions in rows, so they are the operand's major dimension the other way round).
//
// Softmax in one pass.  The sum refers to a maximum m of the row's scores and O to a of its s + log2 vs, both only moved when
// outgrown by more than 6 (log2), so O is rarely rescaled (2 instead of 6: 4096 tokens 251 us instead of 244).
// Weights enter as e^s vs / 2^a * 2^9, below 2^15: f16 keeps 2^-11 of a weight.
//
// The codes, exact in f16, are what is multiplied; ks enters at the score and vs at the weight, in float32.  Multiplied
// into the f16 keys and values instead, once a code and not once a score, they make the weights 1.75 instructions a score
// shorter (4096 tokens 200 us instead of 242), but every product is then rounded to 2^-11: a weight behind a score of 300
// is off by a tenth.
//
// Only what a row sees decides its references.  In a tile of positions whose vs lie within 2^10 of one another the row's largest
// score plus log2 of the tile's largest vs does for a, at most 10 too much: f16 keeps all bits of a weight down to 2^-13 of the
// largest, and 2^-24 of the largest below; in other tiles a is found position by position, and a weight has an exponential of
// its own.  A value whose scale is not finite is zero there, and the rows that see it are marked, so that no row sees NaN
// times zero.
//
// 4096 tokens of 32 heads over 8: 244 us, 0.56 PFLOP/s (33 % of the measured rate); 1152 tokens behind 31616: 0.69 (41 %).  There a
// chain of waits bounds it, not one unit: tensor pipe 25 % busy, issue slots 41 %, exponentials 28 %, the shared memory's
// pipe 58 % (a quarter of it bank conflicts of the converting warps), eight warps with weights waiting for TMEM and for scales.
constexpr int LG_ROWS = 128, LG_POS = 128, LG_THREADS = 17 * 32;
constexpr float LG_SLACK = 6.0f;     // log2: the weights' factor 2^9 leaves these octaves to f16's 65504

struct LongFlags {                   // of a tile of positions, 32 to a warp
    uint32_t there[4];               // which of them are
    uint32_t bad[4];                 // whose value's scale is not finite
    uint32_t big[4];                 // whose key's scale is above 2^90
    uint32_t wide[4];                // whose value's scale is below 2^-10 of the tile's largest
    uint32_t all;                    // are there, and none of them bad
    float v_log, v_unit;             // log2 of a power of two that no value's scale exceeds, and of the unit of those in VW
};
template <int HD> struct LongSmem {
    static constexpr int TILE = LG_ROWS * HD * 2;        // 128 rows of f16, in halves of 64 dimensions
    static constexpr int Q = 0, K = 2 * TILE, V = K + 2 * TILE, RAW = V + 2 * TILE, SC = RAW + 2 * (TILE / 2);
    static constexpr int STAGES = 2, KS = 0, VW = 512, SCALES = 1024;    // of a tile of positions: ks [128], vs / 2^v_unit [128]
    static constexpr int BYTES = SC + STAGES * SCALES;
    static_assert(BYTES + 1024 <= 227 * 1024, "with the static shared memory, which starts the dynamic part on 1024 bytes");
};

__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 lanes x 32 consecutive columns of TMEM -> 32 registers a thread.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
// Pairs of floats in one instruction.
__device__ __forceinline__ float2 pair_op(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)), "l"(reinterpret_cast<unsigned long long &>(c)));
    return r;
}
__device__ __forceinline__ float2 pair_mul(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
__device__ __forceinline__ float2 pair_add(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
// Shared-memory descriptor of an operand whose major dimension is not the summed one (values: rows are positions, which are
// summed over, 64 dimensions of f16 to a 128-byte row, 128-byte swizzle): 8 rows are 1024 bytes (stride offset), the
// next 64 dimensions `half_bytes` further (leading offset).
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t half_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
    d |= (uint64_t)(half_bytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// Where 16-byte chunk c (8 f16) of row `row` of a 128-row tile lies: halves of 64 dimensions, 128-byte swizzle.
__device__ __forceinline__ int f16_chunk_at(int row, int c) { return (c >> 3) * (128 * 128) + row * 128 + 16 * ((c & 7) ^ (row & 7)); }

template <int HD>
__global__ void __launch_bounds__(LG_THREADS, 1)
attention_quant_long_kernel(const AttnQuant p, int skip_short, int span, uint32_t polls) {
    using Sm = LongSmem<HD>;
    constexpr int CH = HD / 16;                          // 16-byte chunks of codes in a row
    extern __shared__ __align__(1024) uint8_t lg_smem[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[Sm::STAGES], sc_empty[Sm::STAGES], s_full[2], p_full[2], o_full[2];
    __shared__ LongFlags flags_s[Sm::STAGES];
    __shared__ uint32_t tmem_base_s, look_s[2][4];
    __shared__ float top_s[2][4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&k_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 128);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < Sm::STAGES; i++) {
            mbar_init(&sc_full[i], 256);
            mbar_init(&sc_empty[i], 8);
        }
        mbar_init_fence();
    }
    pdl_prologue();
    // ---- which rows (span: 256, or 128 for tile 0 alone): blocks of the requests in order, of a request the last (longest) ones first, KV heads innermost ----
    const int group = p.n_heads / p.n_kv, kvh = blockIdx.x % p.n_kv;
    int want = blockIdx.x / p.n_kv, req = -1;
    Request r = {0, 0, 0};
    for (int q0 = 0; q0 < p.num_req && req < 0; q0 += 32) {
        Request mine = {0, 0, 0};
        int blocks = 0;
        if (q0 + lane < p.num_req) {
            mine = request_of(p, q0 + lane);
            const long long rows = (long long)mine.count * group;
            blocks = skip_short && rows <= SHORT_ROWS ? 0 : (int)((rows + span - 1) / span);
        }
        int inc = blocks;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want < inc);
        if (hit) {
            const int src = __ffs(hit) - 1;
            req = q0 + src;
            r.first = __shfl_sync(0xffffffffu, mine.first, src);
            r.count = __shfl_sync(0xffffffffu, mine.count, src);
            r.before = __shfl_sync(0xffffffffu, mine.before, src);
            want = __shfl_sync(0xffffffffu, inc, src) - 1 - want;
        } else {
            want -= __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    if (req < 0) return;                                 // the grid holds as many CTAs as any batch of this size can need
    const int row0 = want * span, rows = min(r.count * group - row0, span);      // of this CTA: 1 .. 256
    // positions that tile t's last row sees, and tiles of positions
    int nt[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int n = min(rows - t * LG_ROWS, LG_ROWS);
        const int end = n > 0 ? r.before + (row0 + t * LG_ROWS + n - 1) / group + 1 : 0;
        nt[t] = end > 0 ? (end + LG_POS - 1) / LG_POS : 0;
    }
    const int n_tiles = max(nt[0], nt[1]);               // tile 1's rows come later and see more, if there are any
    const int kv_end = r.before + (row0 + rows - 1) / group + 1;
    if (warp == 16) { tmem_alloc(&tmem_base_s, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;                   // scores of tile t at 128 t, O at 256 + 128 t
    bool dead = false;
    // A whole warp: gives up once; then nothing is waited for any more.  Lanes leave the polling each for itself, and what follows
    // (tcgen05.ld / st, bar.sync) is .aligned: the warp has to have met again.
    auto wait = [&](uint64_t *bar, uint32_t parity, uint32_t code) {
        if (!dead && !mbar_wait(bar, parity, polls)) { dead = true; report_error(p.err, code); }
        __syncwarp();
    };

    if (warp < 8) {
        // ================= weights =================
        const int t = warp >> 2, i = tid & 127, rr = row0 + t * LG_ROWS + i;
        const bool on = t * LG_ROWS + i < rows;
        const int len = on ? r.before + rr / group + 1 : 0;
        const int min_len = r.before + (row0 + t * LG_ROWS) / group + 1;         // what the tile's first row sees
        const size_t off = on ? ((size_t)(r.first + rr / group) * p.n_heads + (size_t)kvh * group + rr % group) * HD : 0;
        // the row of queries: its size, then scaled by a power of two to f16 and into the operand's layout
        float amax = 0.0f;
        const uint16_t *q = (const uint16_t *)p.q + off;
#pragma unroll 8
        for (int c = 0; c < HD / 8; c++) {
            const uint4 u = on ? *reinterpret_cast<const uint4 *>(q + 8 * c) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int x = 0; x < 4; x++) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xFFFF0000u))));
        }
        const int ex = row_exponent(amax);
        const float up = exp2i(ex), c_row = exp2i(-ex) * (1.4426950408889634f / sqrtf((float)HD));
#pragma unroll 8
        for (int c = 0; c < HD / 8; c++) {
            const uint4 u = on ? *reinterpret_cast<const uint4 *>(q + 8 * c) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            uint32_t h[4];
#pragma unroll
            for (int x = 0; x < 4; x++) h[x] = pack_f16(__uint_as_float(w[x] << 16) * up, __uint_as_float(w[x] & 0xFFFF0000u) * up);
            *reinterpret_cast<uint4 *>(lg_smem + Sm::Q + t * Sm::TILE + f16_chunk_at(i, c)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&q_full[t]);

        const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);          // this warp's 32 lanes
        const uint32_t s_col = lane_base + 128 * t, o_col = lane_base + 256 + 128 * t;
        float m_ref = -INFINITY, a_ref = -INFINITY, l = 0.0f;            // the sum counts in 2^m_ref, O in 2^(a_ref - 9)
        for (int j = 0; j < n_tiles; j++) {
            const int st = j % Sm::STAGES;
            wait(&sc_full[st], (j / Sm::STAGES) & 1, KERR_FULL_WAIT);
            if (j < nt[t]) {
                const uint8_t *sc = lg_smem + Sm::SC + st * Sm::SCALES;
                const float *ks = reinterpret_cast<const float *>(sc + Sm::KS), *vw = reinterpret_cast<const float *>(sc + Sm::VW);
                const LongFlags &fl = flags_s[st];
                const bool wide = (fl.wide[0] | fl.wide[1] | fl.wide[2] | fl.wide[3] | fl.big[0] | fl.big[1] | fl.big[2] | fl.big[3]) != 0;
                const bool masked = (j + 1) * LG_POS > min_len || fl.all == 0 || wide;     // (rows past the end do what the others do, for nothing)
                wait(&s_full[t], j & 1, KERR_MMA_WAIT);
                tc_fence_after();
                auto bits_of = [&](int c) -> uint32_t {  // which of the 32 positions of chunk c this row sees
                    const int n = len - j * LG_POS - 32 * c;
                    const uint32_t there = fl.there[c];
                    return n <= 0 ? 0u : n >= 32 ? there : there & ((1u << n) - 1);
                };
                // Three forms of the code, chosen by the warp: most tiles are seen by every row whole, and a test a score costs
                // more than the score's own arithmetic (MASKED); scales that differ by much are rare (WIDE).  Each 16 columns are
                // asked for while the 16 before are worked on.  (Unrolled whole, or with weights stored 16 registers at a time,
                // registers are spilled: 4096 tokens 252 us instead of 245.)
                uint32_t v[2][16];
                const float2 c2 = make_float2(c_row, c_row);
                float mx = -INFINITY, mv = -INFINITY;    // of what the row sees: the largest score, at least the largest s + log2 vs
                auto largest = [&](auto mask_tag, auto wide_tag) {
                    constexpr bool MASKED = decltype(mask_tag)::value, WIDE = decltype(wide_tag)::value;
                    float mx1 = -INFINITY, mv1 = -INFINITY;
                    tmem_ld16(s_col, v[0]);
                    tmem_ld_wait();
#pragma unroll (MASKED ? 1 : 2)
                    for (int cc = 0; cc < 4; cc++) {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const int c = 2 * cc + half;
                            const uint32_t(&u)[16] = v[half];
                            tmem_ld16(s_col + 16 * ((c + 1) & 7), v[half ^ 1]);       // after the last one the first again, for the weights
                            uint32_t bits = 0;
                            if constexpr (MASKED) bits = bits_of(c >> 1) >> (16 * (c & 1));
#pragma unroll
                            for (int x = 0; x < 16; x += 4) {
                                const float4 k4 = *reinterpret_cast<const float4 *>(ks + 16 * c + x);
                                float2 ka = make_float2(k4.x, k4.y), kb = make_float2(k4.z, k4.w);
                                if constexpr (WIDE) {        // a sum of codes and queries, below 2^30, times a scale of 2^98 would leave float32
                                    ka = pair_mul(ka, c2);
                                    kb = pair_mul(kb, c2);
                                }
                                float2 a = pair_mul(make_float2(__uint_as_float(u[x]), __uint_as_float(u[x + 1])), ka);
                                float2 d = pair_mul(make_float2(__uint_as_float(u[x + 2]), __uint_as_float(u[x + 3])), kb);
                                if constexpr (MASKED) {
                                    if (!(bits >> x & 1)) a.x = -INFINITY;
                                    if (!(bits >> (x + 1) & 1)) a.y = -INFINITY;
                                    if (!(bits >> (x + 2) & 1)) d.x = -INFINITY;
                                    if (!(bits >> (x + 3) & 1)) d.y = -INFINITY;
                                }
                                if constexpr (WIDE) {
                                    const float4 w4 = *reinterpret_cast<const float4 *>(vw + 16 * c + x);
                                    auto share = [&](float score, float vs) { return vs == 0.0f ? -INFINITY : score + log2_of(power_above(fabsf(vs))); };
                                    mv = fmaxf(mv, fmaxf(share(a.x, w4.x), share(a.y, w4.y)));
                                    mv1 = fmaxf(mv1, fmaxf(share(d.x, w4.z), share(d.y, w4.w)));
                                }
                                mx = fmaxf(mx, fmaxf(a.x, a.y));
                                mx1 = fmaxf(mx1, fmaxf(d.x, d.y));
                            }
                            tmem_ld_wait();
                        }
                    }
                    mx = fmaxf(mx, mx1);
                    if constexpr (!WIDE) mx *= c_row;
                    mv = WIDE ? fmaxf(mv, mv1) + fl.v_unit : mx + fl.v_log;
                };
                if (!masked) largest(std::false_type{}, std::false_type{});
                else if (!wide) largest(std::true_type{}, std::false_type{});
                else largest(std::true_type{}, std::true_type{});
                // ---- move the references, O and the sum where they have been outgrown ----
                const float m_new = mx > m_ref + LG_SLACK ? mx : m_ref, a_new = mv > a_ref + LG_SLACK ? mv : a_ref;      // -inf: by any at all
                const float m_base = m_new == -INFINITY ? 0.0f : m_new, a_base = a_new == -INFINITY ? 0.0f : a_new;
                if (m_new != m_ref) l *= ex2(m_ref - m_base);
                if (j > 0 && __any_sync(0xffffffffu, a_new != a_ref)) {
                    const float f = a_new == a_ref ? 1.0f : ex2(a_ref - a_base);
#pragma unroll
                    for (int c = 0; c < HD / 16; c++) {
                        uint32_t o[16];
                        tmem_ld16(o_col + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tmem_st16(o_col + 16 * c, o);
                    }
                }
                m_ref = m_new;
                a_ref = a_new;
                // ---- the weights, over the scores ----
                const float from = a_base - (9.0f + fl.v_unit);          // what the exponents of weights count from
                // One exponential for weight and sum, unless what the sum gets would leave float32 below.
                const bool apart = wide || __any_sync(0xffffffffu, from - m_base > 80.0f);
                auto weights = [&](auto mask_tag, auto apart_tag) {
                    constexpr bool MASKED = decltype(mask_tag)::value, APART = decltype(apart_tag)::value;
                    const float2 nb = make_float2(-from, -from);
                    float2 l2 = make_float2(0.0f, 0.0f);
                    bool bad = false;
                    uint32_t w[8];
#pragma unroll (MASKED ? 1 : 2)
                    for (int cc = 0; cc < 4; cc++) {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const int c = 2 * cc + half;
                            const uint32_t(&u)[16] = v[half];
                            if (c < 7) tmem_ld16(s_col + 16 * (c + 1), v[half ^ 1]);
                            uint32_t bits = 0;
                            if constexpr (MASKED) {
                                bits = bits_of(c >> 1);
                                bad |= (bits & fl.bad[c >> 1]) != 0;
                                bits >>= 16 * (c & 1);
                            }
#pragma unroll
                            for (int x = 0; x < 16; x += 4) {
                                const float4 k4 = *reinterpret_cast<const float4 *>(ks + 16 * c + x), w4 = *reinterpret_cast<const float4 *>(vw + 16 * c + x);
#pragma unroll
                                for (int y = 0; y < 2; y++) {
                                    const int at = x + 2 * y;
                                    const float2 s2 = make_float2(__uint_as_float(u[at]), __uint_as_float(u[at + 1]));
                                    const float2 k2 = y ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y), v2 = y ? make_float2(w4.z, w4.w) : make_float2(w4.x, w4.y);
                                    float2 e, z;             // what the sum gets, the weights
                                    if constexpr (APART) {
                                        const float2 score = pair_mul(s2, pair_mul(k2, c2));
                                        e = make_float2(ex2(score.x - m_base), ex2(score.y - m_base));
                                        const uint32_t px = power_of(fabsf(v2.x)), py = power_of(fabsf(v2.y));       // vs = 2^p times its rest
                                        z.x = ex2((score.x - from) + log2_of(px)) * (v2.x * __uint_as_float((254u << 23) - px));
                                        z.y = ex2((score.y - from) + log2_of(py)) * (v2.y * __uint_as_float((254u << 23) - py));
                                    } else {
                                        e = pair_op(pair_mul(s2, k2), c2, nb);
                                        e = make_float2(ex2(e.x), ex2(e.y));
                                    }
                                    if constexpr (MASKED) {
                                        if (!(bits >> at & 1)) e.x = z.x = 0.0f;
                                        if (!(bits >> (at + 1) & 1)) e.y = z.y = 0.0f;
                                    }
                                    l2 = pair_add(l2, e);
                                    if constexpr (!APART) z = pair_mul(e, v2);
                                    w[at / 2] = pack_f16(z.x, z.y);
                                }
                            }
                            if (c < 7) tmem_ld_wait();
                            tmem_st8(s_col + 8 * c, w);
                        }
                    }
                    l += APART ? l2.x + l2.y : (l2.x + l2.y) * ex2(from - m_base);
                    if (MASKED && bad) l = __int_as_float(0x7FC00000);   // sees a value that is NaN
                };
                if (apart) weights(std::true_type{}, std::true_type{});
                else if (masked) weights(std::true_type{}, std::false_type{});
                else weights(std::false_type{}, std::false_type{});
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_empty[st]);
            __syncwarp();
        }
        // ---- O, divided by the sum ----
        // 2^(a - 9 - m) / l in two factors: each stays in float32's range
        const float back = (a_ref - m_ref) - 9.0f, back0 = truncf(0.5f * back);
        const bool none = a_ref == -INFINITY && l == l;  // nothing seen, or only values of zero
        const float norm0 = none ? 0.0f : ex2(back0), norm1 = none ? 0.0f : ex2(back - back0) / l;
        uint16_t *out = (uint16_t *)p.out + off;
        if (nt[t] > 0) {
            wait(&o_full[t], 0, KERR_MMA_WAIT);
            tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
            uint32_t v[32];
            if (nt[t] > 0) {
                tmem_ld32(o_col + 32 * c, v);
                tmem_ld_wait();
            }
            if (on) {                                    // not so for all lanes of a warp that the rows end in
#pragma unroll
                for (int x = 0; x < 32; x += 8) {
                    uint32_t h[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        // rows without positions: zeros (their columns of O may never have been written)
                        const float a = len > 0 ? __uint_as_float(v[x + 2 * y]) * norm0 * norm1 : 0.0f, b = len > 0 ? __uint_as_float(v[x + 2 * y + 1]) * norm0 * norm1 : 0.0f;
                        const __nv_bfloat162 z = __floats2bfloat162_rn(a, b);
                        h[y] = *reinterpret_cast<const uint32_t *>(&z);
                    }
                    *reinterpret_cast<uint4 *>(out + 32 * c + x) = make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            __syncwarp();
        }
        tc_fence_before();
    } else if (warp < 16) {
        // ================= keys (warps 8-11), values (12-15) =================
        const bool keys = warp < 12;
        const int w = warp & 3;                          // this warp's positions are 32 w .. 32 w + 31 of a tile
        const size_t kv_dim = (size_t)p.n_kv * HD;
        const uint32_t *table = p.block_table + (size_t)req * p.max_blocks;
        const uint8_t *pool = (keys ? p.k_pool : p.v_pool) + (size_t)kvh * HD;
        const float *scales = (keys ? p.k_scales : p.v_scales) + (size_t)kvh * p.num_slots;
        constexpr int RPI = 32 / CH, N = 32 / RPI;       // rows a pass, passes
        const int c = lane % CH;
        uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
        uint8_t *tiles = lg_smem + (keys ? Sm::K : Sm::V), *raw = lg_smem + Sm::RAW + (keys ? 0 : Sm::TILE / 2) + w * 32 * HD;
        float scale_next = 0.0f;
        uint32_t there_next = 0, page = 0;
        auto page_of = [&](int j) -> uint32_t {
            const int pos = j * LG_POS + 32 * w + lane;
            return pos < kv_end ? table[pos / p.block_size] : 0u;
        };
        // The codes travel to shared memory as they are, a tile ahead; the thread that asked for 16 of them converts them, so
        // nobody else waits for them.  Lane x looks up position 32 w + x, and has its scale.
        auto ask = [&](int j) {
            const int pos = j * LG_POS + 32 * w + lane;
            const unsigned long long s64 = (unsigned long long)page * p.block_size + (unsigned)(pos % p.block_size);
            const bool ok = pos < kv_end && s64 < p.num_slots;
            if (pos < kv_end && !ok) report_error(p.err, KERR_SLOT_RANGE);
            const uint32_t slot = ok ? (uint32_t)s64 : 0u;
            there_next = __ballot_sync(0xffffffffu, ok);
            scale_next = ok ? __ldg(scales + slot) : 0.0f;
#pragma unroll
            for (int x = 0; x < N; x++) {
                const int row = x * RPI + lane / CH;
                const size_t at = (size_t)__shfl_sync(0xffffffffu, slot, row) * kv_dim + 16 * c;
                copy16_or_zero(raw + row * HD + 16 * c, pool + at, there_next >> row & 1);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            page = page_of(j + 1);
        };
        if (n_tiles > 0) {
            page = page_of(0);
            ask(0);
        }
        for (int j = 0; j < n_tiles; j++) {
            const int b = j & 1, st = j % Sm::STAGES;
            const uint32_t there = there_next;
            const bool ok = keys || fabsf(scale_next) <= 3.402823466e38f;       // a value's scale that is NaN or infinite: zeros, and marked
            const float scale = ok ? scale_next : 0.0f;
            auto publish = [&]() {
                uint8_t *sc = lg_smem + Sm::SC + st * Sm::SCALES;
                LongFlags &fl = flags_s[st];
                if (keys) {
                    const uint32_t big = __ballot_sync(0xffffffffu, fabsf(scale) > 0x1p90f);
                    if (j >= Sm::STAGES) wait(&sc_empty[st], ((j / Sm::STAGES) & 1) ^ 1, KERR_EMPTY_WAIT);
                    reinterpret_cast<float *>(sc + Sm::KS)[32 * w + lane] = scale;
                    if (lane == 0) {
                        fl.there[w] = there;
                        fl.big[w] = big;
                    }
                } else {
                    float top = fabsf(scale);
#pragma unroll
                    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const uint32_t bad = __ballot_sync(0xffffffffu, !ok);
                    if (lane == 0) {
                        top_s[b][w] = top;
                        look_s[b][w] = there != 0xFFFFFFFFu || bad;      // positions past kv_end, on a page beyond the pool, or marked
                    }
                    __syncwarp();
                    named_barrier_sync(2, 128);          // what the four warps have found
                    const uint32_t most = power_above(fmaxf(fmaxf(top_s[b][0], top_s[b][1]), fmaxf(top_s[b][2], top_s[b][3])));
                    const uint32_t unit = min(most, 127u << 23);         // small values are made larger; larger ones would push others below
                    const uint32_t wide = __ballot_sync(0xffffffffu, ok && (there >> lane & 1) && fabsf(scale) < __uint_as_float(most) * 0x1p-10f);
                    if (j >= Sm::STAGES) wait(&sc_empty[st], ((j / Sm::STAGES) & 1) ^ 1, KERR_EMPTY_WAIT);
                    reinterpret_cast<float *>(sc + Sm::VW)[32 * w + lane] = scale * __uint_as_float((254u << 23) - unit);
                    if (lane == 0) {
                        fl.bad[w] = bad;
                        fl.wide[w] = wide;
                    }
                    if (w == 0 && lane == 0) {
                        fl.all = !(look_s[b][0] | look_s[b][1] | look_s[b][2] | look_s[b][3]);
                        fl.v_log = log2_of(most);
                        fl.v_unit = log2_of(unit);
                    }
                }
                mbar_arrive(&sc_full[st]);
            };
            if (!keys) publish();                        // the weights wait for the scales, the keys' product for the keys
            if (j >= 2) wait(&empty[b], ((j >> 1) & 1) ^ 1, KERR_EMPTY_WAIT);
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            uint8_t *tile = tiles + b * Sm::TILE;
#pragma unroll
            for (int x = 0; x < N; x++) {
                const int row = x * RPI + lane / CH;
                const uint4 u = *reinterpret_cast<const uint4 *>(raw + row * HD + 16 * c);
                uint32_t h[8];
                codes_to_f16(u.x, h[0], h[1]);
                codes_to_f16(u.y, h[2], h[3]);
                codes_to_f16(u.z, h[4], h[5]);
                codes_to_f16(u.w, h[6], h[7]);
                *reinterpret_cast<uint4 *>(tile + f16_chunk_at(32 * w + row, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4 *>(tile + f16_chunk_at(32 * w + row, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&full[b]);
            if (j + 1 < n_tiles) ask(j + 1);
            if (keys) publish();
        }
    } else {
        // ================= products =================
        constexpr uint32_t QK_DESC = umma_idesc_f16(LG_POS);             // N = 128 positions, K-major both
        constexpr uint32_t PV_DESC = umma_idesc_f16(HD) | (1u << 16);    // N = head_dim; the values' major dimension is N
        const uint32_t base = smem_u32(lg_smem);
        const bool one = elect_one();
        auto scores = [&](int t, int j) {
            if (one && !dead) {
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t step = (k >> 2) * (128 * 128) + (k & 3) * 32;
                    umma_f16_ss(tmem + 128 * t, umma_desc_sw128(base + Sm::Q + t * Sm::TILE + step),
                                umma_desc_sw128(base + Sm::K + (j & 1) * Sm::TILE + step), QK_DESC, k > 0);
                }
                umma_commit(&s_full[t]);
            }
            __syncwarp();
        };
        for (int t = 0; t < 2; t++) wait(&q_full[t], 0, KERR_FULL_WAIT);
        if (n_tiles > 0) {
            wait(&k_full[0], 0, KERR_FULL_WAIT);
            tc_fence_after();
            for (int t = 0; t < 2; t++)
                if (nt[t] > 0) scores(t, 0);
            if (one && !dead) umma_commit(&k_empty[0]);
            __syncwarp();
        }
        for (int j = 0; j < n_tiles; j++) {
            wait(&v_full[j & 1], (j >> 1) & 1, KERR_FULL_WAIT);
            if (j + 1 < n_tiles) wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, KERR_FULL_WAIT);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                if (j >= nt[t]) continue;
                wait(&p_full[t], j & 1, KERR_MMA_WAIT);
                tc_fence_after();
                if (one && !dead) {
#pragma unroll
                    for (int k = 0; k < LG_POS / 16; k++)
                        umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k,
                                    umma_desc_sw128_mn(base + Sm::V + (j & 1) * Sm::TILE + k * 2048, 128 * 128), PV_DESC, j > 0 || k > 0);
                    if (j + 1 == nt[t]) umma_commit(&o_full[t]);
                }
                __syncwarp();
                if (j + 1 < nt[t]) scores(t, j + 1);
            }
            if (one && !dead) {
                umma_commit(&v_empty[j & 1]);
                if (j + 1 < n_tiles) umma_commit(&k_empty[(j + 1) & 1]);
            }
            __syncwarp();
        }
        // nothing of this warp's may be under way when the memory goes: the last commits have arrived
        if (n_tiles > 0) mbar_wait(&v_empty[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, polls);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD>
cudaError_t launch_long(const AttnQuant &p, int skip_short, int sm_count, uint32_t polls, cudaStream_t s, bool pdl) {
    // 256 rows a CTA, so that two tiles share keys and values and hide each other's waits; one tile of 128 where that is about
    // a CTA an SM or less (1.25: requests differ in length).  128 tokens of 32 heads over 8: 12.2 us with one tile, 17.0 with
    // two; 128 behind 8064: 187 and 227; 12 chunks of up to 500 tokens, 2 KV heads: 78 and 93; but 1152 tokens: 45.9 and 44.0.
    const long long rows = (long long)p.total_q * (p.n_heads / p.n_kv);
    const int span = rows * p.n_kv <= (long long)sm_count * LG_ROWS * 5 / 4 ? LG_ROWS : 2 * LG_ROWS;
    // every request may end in a block that is not full; the short kernel's, of at most SHORT_ROWS rows, have none
    const long long ends = skip_short && rows / (SHORT_ROWS + 1) < p.num_req ? rows / (SHORT_ROWS + 1) : p.num_req;
    const long long blocks = (rows + span - 1) / span + ends;
    const cudaError_t e = cudaFuncSetAttribute(attention_quant_long_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, LongSmem<HD>::BYTES);
    if (e != cudaSuccess) return e;
    if (blocks * p.n_kv > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    return launch_dependent(attention_quant_long_kernel<HD>, dim3((unsigned)(blocks * p.n_kv)), dim3(LG_THREADS), LongSmem<HD>::BYTES, s, pdl, p,
                            skip_short, span, polls);
}

struct ShortPlan { int rb, terms, hw, per_sm; };
ShortPlan short_plan(const AttnQuant &p, int dtype) {
    const int group = p.n_heads / p.n_kv;
    ShortPlan s;
    // Rows per block: 16 rows cost little more than 8, but a block of 8 leaves registers for nothing to be spilled (64 decode
    // requests: 107 us against 131).  So 8 where that holds what a request has on average, and in batches that mix prompts,
    // the long kernel's, with single tokens; 16 for drafts of a few tokens, and for F32 prompts.
    const double rows = (double)p.total_q * group / p.num_req;
    s.rb = group <= 8 && (rows <= 8 || (rows > SHORT_ROWS && dtype == DT_BF16)) ? 8 : 16;
    s.terms = dtype == DT_F32 ? 2 : 1;
    s.hw = p.n_kv % 4 == 0 ? 4 : p.n_kv % 2 == 0 ? 2 : 1;
    s.per_sm = 2;
    return s;
}
constexpr int SHORT_MAX_GROUPS = 2048;       // head groups of a call
int short_grid(const AttnQuant &p, const ShortPlan &s, int sm_count) {
    const int groups = p.n_kv / s.hw, per = s.per_sm * sm_count / groups;
    return (per < 1 ? 1 : per) * groups;
}
size_t short_workspace(const AttnQuant &p, const ShortPlan &s, int sm_count) {
    return (size_t)short_grid(p, s, sm_count) * 2 * s.hw * s.rb * (p.head_dim + 2) * sizeof(float);
}

constexpr int MERGE_THREADS = 512, MERGE_REQUESTS = 8;       // of attention_quant_merge_kernel
// Few requests, and few rows, since it starts a CTA for each row of the batch, whether or not that was split.
bool merges_after(const AttnQuant &p) { return p.num_req <= MERGE_REQUESTS && p.total_q <= SHORT_ROWS * MERGE_REQUESTS; }
// What the launches of one call share.
struct ShortCall {
    ShortMaps maps;
    int dtype, grid, only_short;
    uint32_t polls;
    float *ws;
    uint32_t *counters;
    bool tma, pdl;
    cudaStream_t stream;
    uint64_t *launches;
};
// Runs of 16 positions stay within a page, and the scales of a KV head start on 16 bytes.
bool tma_fits(const AttnQuant &p) { return p.block_size % 16 == 0 && p.num_slots % 4 == 0; }

cudaError_t encode_maps(const AttnQuant &p, int hw, ShortMaps *m) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)p.head_dim, p.num_slots, (cuuint64_t)p.n_kv};
    const cuuint64_t strides[2] = {(cuuint64_t)p.n_kv * p.head_dim, (cuuint64_t)p.head_dim};
    const cuuint32_t box[3] = {(cuuint32_t)p.head_dim, 16, (cuuint32_t)hw}, step[3] = {1, 1, 1};
    for (int i = 0; i < 2; i++) {
        const CUresult r = enc(i ? &m->v : &m->k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(i ? p.v_pool : p.k_pool), dims,
                               strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               p.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return cudaErrorInvalidValue;
        const cudaError_t e = encode_2d(i ? &m->vs : &m->ks, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, i ? p.v_scales : p.k_scales, p.num_slots,
                                        (uint64_t)p.n_kv, (uint64_t)p.num_slots * 4, 16, (uint32_t)hw, CU_TENSOR_MAP_SWIZZLE_NONE);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <int HD, int RB, int TERMS, int HW, int NST, bool TMA>
cudaError_t launch_short(const AttnQuant &p, const ShortCall &c) {
    constexpr size_t meet = HW == SH_WARPS ? 0 : (size_t)SH_WARPS * RB * (16 + 2) * sizeof(float);
    using St = ShortStage<HD, HW>;
    constexpr size_t smem = NST * (St::BYTES + St::AUX) + meet;
    static_assert(2 * (smem + 2048) <= 228 * 1024, "two CTAs' shared memory");
    auto k = attention_quant_short_kernel<HD, RB, TERMS, HW, NST, TMA>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(k, dim3((unsigned)c.grid), dim3(SH_THREADS + (TMA ? 32 : 128)), smem, c.stream, c.pdl, c.maps, p,
                            (int)(c.dtype == DT_BF16), c.only_short, c.polls, c.ws, c.counters, (int)!merges_after(p));
}
template <int HD, int RB, int TERMS, int NST>
cudaError_t launch_short_hw(const AttnQuant &p, int hw, const ShortCall &c) {
    switch (hw) {
        case 4: return c.tma ? launch_short<HD, RB, TERMS, 4, NST, true>(p, c) : launch_short<HD, RB, TERMS, 4, NST, false>(p, c);
        case 2: return c.tma ? launch_short<HD, RB, TERMS, 2, NST, true>(p, c) : launch_short<HD, RB, TERMS, 2, NST, false>(p, c);
        default: return c.tma ? launch_short<HD, RB, TERMS, 1, NST, true>(p, c) : launch_short<HD, RB, TERMS, 1, NST, false>(p, c);
    }
}
// The parts of one row (query token, head), joined in order: the form for few requests, each in many parts, where a CTA a
// row has more loads under way than the CTAs that happen to be last (one request of 131071 positions, 148 parts a row: 56 us
// in all instead of 66, one of 1000: 12.7 instead of 15.2).  Looking its request up costs a CTA too much where there are many
// (64 requests: 65 us for this kernel beside 97), and there are few parts a row to join then.
template <int HD>
__global__ void __launch_bounds__(MERGE_THREADS)
attention_quant_merge_kernel(const AttnQuant p, int bf16, const Rows rows, int ctas, const float *__restrict__ ws) {
    constexpr int PER = MERGE_THREADS / (HD / 4);        // parts at a time: HD / 4 threads to one
    __shared__ float4 acc_s[MERGE_THREADS];
    __shared__ float red[MERGE_THREADS / 32], lsum[PER];
    const int head = blockIdx.x % p.n_heads, gq = blockIdx.x / p.n_heads, tid = threadIdx.x;
    const int group = p.n_heads / p.n_kv, kvh = head / group;
    pdl_prologue();
    Request r = {0, 0, 0};
    int blocks = 0, tiles = 0;
    long long total = 0, before = 0;
#pragma unroll
    for (int q = 0; q < MERGE_REQUESTS; q++) {
        if (q >= p.num_req) break;
        const Request x = request_of(p, q);
        int b, t;
        shape_of(p, rows, x, b, t);
        if (gq >= x.first && gq < x.first + x.count) { r = x; blocks = b; tiles = t; before = total; }
        total += (long long)b * t;
    }
    if (blocks == 0) return;                             // behind the last request, or the other kernel's
    const int rr = (gq - r.first) * group + head % group, rb = rr / rows.rb, i = rr % rows.rb;
    const int n = sharers(total, ctas), groups = p.n_kv / rows.hw, hg = kvh / rows.hw, hd = kvh % rows.hw;
    const long long item = before + (long long)rb * tiles;
    const int c0 = holder(total, n, item), c1 = holder(total, n, item + tiles - 1);
    if (c0 == c1) return;                                // one CTA had all of it and wrote the row
    const int inside = item > first_unit(total, n, c0) ? 1 : 0;
    const float2 *ml = reinterpret_cast<const float2 *>(ws + (size_t)ctas * groups * 2 * rows.hw * rows.rb * HD);
    auto part = [&](int c) { return ((size_t)((c * groups + hg) * 2 + (c == c0 ? inside : 0)) * rows.hw + hd) * rows.rb + i; };
    float m = -INFINITY;
    for (int c = c0 + tid; c <= c1; c += MERGE_THREADS) m = fmaxf(m, ml[part(c)].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < MERGE_THREADS / 32; w++) m = fmaxf(m, red[w]);
    const float base = m == -INFINITY ? 0.0f : m;
    const int d = 4 * (tid % (HD / 4)), mine = tid / (HD / 4);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int c = c0 + mine; c <= c1; c += PER) {
        const size_t x = part(c);
        const float2 v = ml[x];
        const float4 q = *reinterpret_cast<const float4 *>(ws + x * HD + d);
        const float w = ex2(v.x - base);
        l = fmaf(v.y, w, l);
        acc.x = fmaf(q.x, w, acc.x); acc.y = fmaf(q.y, w, acc.y); acc.z = fmaf(q.z, w, acc.z); acc.w = fmaf(q.w, w, acc.w);
    }
    acc_s[tid] = acc;
    if (d == 0) lsum[mine] = l;
    __syncthreads();
    if (tid >= HD / 4) return;
    l = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int x = 0; x < PER; x++) {
        const float4 q = acc_s[x * (HD / 4) + tid];
        l += lsum[x];
        acc.x += q.x; acc.y += q.y; acc.z += q.z; acc.w += q.w;
    }
    const float norm = l == 0.0f ? 0.0f : 1.0f / l;
    store4(p.out, ((size_t)gq * p.n_heads + head) * HD + d, make_float4(acc.x * norm, acc.y * norm, acc.z * norm, acc.w * norm), bf16);
}

template <int HD>
cudaError_t launch_short_all(const AttnQuant &p, const ShortPlan &pl, const ShortCall &c) {
    constexpr int NST = HD == 128 ? 3 : 5;
    cudaError_t e;
    if (pl.terms == 2) e = pl.rb == 8 ? launch_short_hw<HD, 8, 2, NST>(p, pl.hw, c) : launch_short_hw<HD, 16, 2, NST>(p, pl.hw, c);
    else e = pl.rb == 8 ? launch_short_hw<HD, 8, 1, NST>(p, pl.hw, c) : launch_short_hw<HD, 16, 1, NST>(p, pl.hw, c);
    if (e != cudaSuccess || !merges_after(p)) return e;
    const Rows rows{pl.rb, 16 * SH_TILES / pl.hw, pl.hw, c.only_short};
    ++*c.launches;
    return launch_dependent(attention_quant_merge_kernel<HD>, dim3((unsigned)p.total_q * p.n_heads), dim3(MERGE_THREADS), 0, c.stream, c.pdl,
                            p, (int)(c.dtype == DT_BF16), rows, c.grid / (p.n_kv / pl.hw), (const float *)c.ws);
}

bool mma_supported(const AttnQuant &p) { return (p.head_dim == 64 || p.head_dim == 128) && p.n_kv <= SHORT_MAX_GROUPS; }

}  // namespace

size_t attention_quant_workspace(const AttnQuant &p, int dtype, int sm_count) {
    return mma_supported(p) ? short_workspace(p, short_plan(p, dtype), sm_count) : 0;
}

// Two levels x two parts a CTA; a call with more head groups than resident CTAs has a CTA each.
size_t attention_quant_counter_bytes(int sm_count) { return (size_t)4 * (2 * sm_count > SHORT_MAX_GROUPS ? 2 * sm_count : SHORT_MAX_GROUPS) * sizeof(uint32_t); }

cudaError_t launch_attention_quant(const AttnQuant &p, int dtype, float *ws, uint32_t *counters, int sm_count, uint32_t polls, cudaStream_t s,
                                   bool pdl, uint64_t *launches) {
    if (p.total_q <= 0 || p.num_req <= 0) return cudaSuccess;
    if (!mma_supported(p)) {
        ++*launches;
        return launch_dependent(attention_quant_simple_kernel, dim3((unsigned)p.total_q * p.n_heads), dim3(AQ_TILE), 0, s, pdl, p,
                                (int)(dtype == DT_BF16));
    }
    const ShortPlan pl = short_plan(p, dtype);
    ShortCall c = {};
    c.dtype = dtype; c.grid = short_grid(p, pl, sm_count); c.polls = polls; c.ws = ws; c.counters = counters; c.pdl = pdl; c.stream = s; c.launches = launches;
    c.tma = tma_fits(p);
    if (c.tma) {
        const cudaError_t e = encode_maps(p, pl.hw, &c.maps);
        if (e != cudaSuccess) return e;
    }
    // Requests of more than 16 rows go to the long kernel, the others to the short one, which cuts what it gets into
    // blocks of 16 rows.  The lengths are on the device; the host knows the totals.  As many tokens as requests: a
    // decode batch, all to the short kernel.  One request: one kernel.  F32 has no long kernel.
    const long long rows = (long long)p.total_q * (p.n_heads / p.n_kv);
    const bool decode = p.total_q <= p.num_req || rows <= SHORT_ROWS;
    if (dtype == DT_BF16 && !decode) {
        const int both = p.num_req > 1;
        cudaError_t e = p.head_dim == 128 ? launch_long<128>(p, both, sm_count, polls, s, pdl) : launch_long<64>(p, both, sm_count, polls, s, pdl);
        ++*launches;
        if (e != cudaSuccess || !both) return e;
        c.only_short = 1;
    }
    ++*launches;
    return p.head_dim == 128 ? launch_short_all<128>(p, pl, c) : launch_short_all<64>(p, pl, c);
}

}  // namespace llmrs
