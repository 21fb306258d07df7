// A paged key/value cache held in 4 bits: the writer that quantises new rows into their pages, and
// attention of one or a few new tokens per sequence over it.
//
// Page layout: kv head h of a page has page_tokens * (hd + 8 * groups) bytes at h times that size:
// K codes [page_tokens][hd/2], K parameters [page_tokens][groups] (f16 scale, f16 offset), then V
// the same way.  A group is min(64, hd) neighbouring elements of one token's head; code c stands for
// scale * c + offset, element 2i of a row in the low half of byte i.  72 bytes a token and kv head
// at hd 64, against 256 in f16.  One head of one page is contiguous, so a single bulk copy fetches it.

#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>

#include "enx_internal.cuh"
#include "k_kv4.cuh"

namespace enx {

namespace {

constexpr uint32_t kKvSpin = 1u << 24;  // default limit of a wait, and the limit of the drain waits
__device__ uint32_t g_kv4_spin = kKvSpin;
__device__ uint32_t g_kv4_err = 0;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The smallest and the largest of three, NaN if one is.
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The whole number from 0 to 15 nearest to (x - m) / s, ties to even, where c is within one of it.  Exact: x -
// m is split into its f32 value and the rest (two-sum), and the sign of x - m - (k + 1/2) s, with k + 1/2 the
// border on that side of c on which the value lies, decides; the FMA's result has the sign of the exact one.
__device__ __forceinline__ float nearest_code(float x, float m, float s, float c) {
    const float d = x - m, back = d - x, rest = (x - (d - back)) - (m + back);
    const float side = fmaf(-c, s, d) + rest < 0.f ? -0.5f : 0.5f, at = c + side;
    const float over = fmaf(-at, s, d) + rest;  // how far the value lies above that border
    const bool odd = (int)c & 1, beyond = side > 0.f ? over > 0.f : over < 0.f;
    return fminf(fmaxf(beyond || (over == 0.f && odd) ? c + 2.f * side : c, 0.f), 15.f);
}

struct WriteArgs {
    const void *k, *v;
    void *k_out, *v_out;  // contiguous [tokens][kv_heads][hd], or null
    long long k_token, k_head, v_token, v_head;  // strides in elements
    uint8_t* pool;
    const int32_t *table, *seqs, *positions;
    const int32_t* lengths;  // or null: positions are taken as they are
    uint32_t tokens, rows, width, pages, page_shift, kv_heads, hd, head_shift;
    int vec;  // all rows start on 16 bytes
};

}  // namespace

// Eight elements per thread, 4 (hd 32) or 8 threads per group.  HBM-bound: rows in, codes and the
// values they stand for out.  The f16 scale and the codes are decided exactly: quotients are taken
// in f32, and settled without rounding where f32 cannot tell on which side of a border they lie.  A group with
// an element that is not finite gets NaN parameters, so that what reads it is not finite either.
//
// What it costs otherwise is instructions: K and V of a place share the search for it, rounding and packing
// are additions and FMAs, not conversions and shifts, and the rows are fetched while their place is still
// looked up.
// 41 thousand tokens of 8 heads of 128 in bf16: 105 us, 3.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) k_kv4_write(WriteArgs a) {
    // thread = 8 elements of one token and head, of K and of V
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;  // below 2^32: the host refuses more
    const uint32_t row = item >> a.head_shift, e8 = item & (a.hd / 8 - 1);
    const uint32_t token = row / a.kv_heads, head = row - token * a.kv_heads;
    bool live = token < a.tokens;
    alignas(16) T raw[2][8];
    int32_t pos = -1, seq = -1, page = -1;
    if (live) {
        pos = a.positions[token];
        seq = a.seqs[token];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const T* src = static_cast<const T*>(kv ? a.v : a.k) + (long long)token * (kv ? a.v_token : a.k_token) +
                           (long long)head * (kv ? a.v_head : a.k_head) + e8 * 8;
            if (a.vec) {
#pragma unroll
                for (uint32_t i = 0; i < sizeof(T) / 2; ++i)
                    reinterpret_cast<uint4*>(raw[kv])[i] = ld_stream(reinterpret_cast<const uint4*>(src) + i);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[kv][i] = src[i];
            }
        }
        if (pos >= 0 && seq >= 0 && (uint32_t)seq < a.rows && ((uint32_t)pos >> a.page_shift) < a.width &&
            (!a.lengths || pos < a.lengths[seq]))
            page = a.table[(size_t)seq * a.width + ((uint32_t)pos >> a.page_shift)];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i / 8][i % 8] = from_f<T>(0.f);
    }
    live = page >= 0 && (uint32_t)page < a.pages;
    const uint32_t lanes = a.hd < 64 ? 4 : 8;  // of a group (whole groups lie in a warp)
    const uint32_t groups = a.hd > 64 ? a.hd / 64 : 1, pt = 1u << a.page_shift, slot = (uint32_t)pos & (pt - 1);
    const uint32_t head_bytes = pt * (a.hd + 8 * groups);
    uint8_t* at = a.pool + ((size_t)(uint32_t)max(page, 0) * a.kv_heads + head) * head_bytes;
    const size_t back_at = ((size_t)token * a.kv_heads + head) * a.hd + e8 * 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(raw[kv][i]);
        float lo = min3(min3(min3(x[0], x[1], x[2]), x[3], x[4]), min3(x[5], x[6], x[7]), x[0]);
        float hi = max3(max3(max3(x[0], x[1], x[2]), x[3], x[4]), max3(x[5], x[6], x[7]), x[0]);
#pragma unroll
        for (uint32_t o = 1; o < 8; o <<= 1)
            if (o < lanes) {
                const float l = __shfl_xor_sync(0xffffffffu, lo, o), h = __shfl_xor_sync(0xffffffffu, hi, o);
                lo = min3(lo, l, l);
                hi = max3(hi, h, h);
            }
        if (!live) continue;
        __half sc, of;
        if (fabsf(lo) < INFINITY && fabsf(hi) < INFINITY) {  // (both are NaN where an element is)
            // the f32 quotient is off by less than 2^-21 of itself (difference, product, 1/15)
            const float q = (hi - lo) * (1.f / 15.f);
            sc = __float2half_rn(fminf(q * (1.f - 0x1p-20f), 65504.f));
            if (__half_as_ushort(sc) != __half_as_ushort(__float2half_rn(fminf(q * (1.f + 0x1p-20f), 65504.f))))
                sc = __float2half_rn((float)fmin(((double)hi - (double)lo) / 15.0, 65504.0));
            of = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
        } else {
            sc = of = __ushort_as_half(0x7e00);  // NaN
        }
        const float s = __half2float(sc), m = __half2float(of);
        const float inv15 = s > 0.f ? __fdividef(1.f / 15.f, s) : 0.f;  // 0: every code is 0
        constexpr float kWhole = 12582912.f;                             // 1.5 * 2^23: added, it rounds to whole numbers
        float c[8], val[8];
        bool border = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float u = __saturatef((x[i] - m) * inv15);  // the code before rounding, in fifteenths
            c[i] = fmaf(u, 15.f, kWhole) - kWhole;
            // 15 u is off by less than 15 * 6 * 2^-24 < 2^-17 (difference, quotient of 2 ulp, 1/15, product, FMA);
            // borders are at c +- 1/2
            border = border || fabsf(fmaf(u, 15.f, -c[i])) > 0.5f - 0x1p-16f;
        }
        if (border) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (s > 0.f) c[i] = nearest_code(x[i], m, s, c[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) val[i] = fmaf(s, c[i], m);
        // four codes at a time are a whole number below 2^16, exactly
        const float w0 = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]) + 8388608.f;
        const float w1 = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]) + 8388608.f;
        const uint32_t word = __byte_perm(__float_as_uint(w0), __float_as_uint(w1), 0x5410);
        uint8_t* half = at + (kv ? head_bytes / 2 : 0);
        *reinterpret_cast<uint32_t*>(half + slot * (a.hd / 2) + e8 * 4) = word;
        if ((e8 & (lanes - 1)) == 0)
            *reinterpret_cast<__half2*>(half + pt * (a.hd / 2) + (slot * groups + (lanes == 8 ? e8 >> 3 : 0)) * 4) = __halves2half2(sc, of);
        T* back = static_cast<T*>(kv ? a.v_out : a.k_out);
        if (back) {
            alignas(16) T tmp[8];
            // 15 steps of a scale that was rounded up may pass f16's largest number: it saturates here as there
            if (std::is_same<T, __half>::value && fmaf(s, 15.f, m) > 65504.f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) val[i] = fminf(val[i], 65504.f);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) tmp[i] = from_f<T>(val[i]);
            if (a.vec) {
#pragma unroll
                for (uint32_t i = 0; i < sizeof(T) / 2; ++i)
                    reinterpret_cast<uint4*>(back + back_at)[i] = reinterpret_cast<const uint4*>(tmp)[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) back[back_at + i] = tmp[i];
            }
        }
    }
}

// ---- attention ----------------------------------------------------------------------------------

namespace {

constexpr uint32_t kKvChunk = 64;  // tokens of a stage and of a unit of work
constexpr uint32_t kKvStages = 2;  // per warp: one is computed on while the other lands
constexpr uint32_t kKvWarps = 4;
constexpr uint32_t kKvMinRun = 1;  // units a warp takes at least (2 and 4 cost short calls 1 to 4 us and gain nothing)
constexpr float kKvLow = -1e30f;   // a row's reference before it has seen a score

struct AttnArgs {
    const void* q;
    long long q_seq, q_query, q_head;  // strides in elements
    const uint8_t* pool;
    const int32_t *table, *lengths, *seqs;  // seqs may be null: row b is sequence b
    void* out;                              // [batch][queries][heads][hd]
    uint32_t* head_ws;                      // units before each sequence [batch + 1], units per run
    float* part;                            // partials: [2 * runs][8 NT][hd + 4]: sums, then m, l
    uint32_t batch, queries, heads, kv_heads, rows, width, pages, page_shift, tiles, most_chunks;
    float scale_log2;  // the softmax scale times log2(e)
    int vec;           // q's rows start on 16 bytes
};

__device__ __forceinline__ uint32_t su32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(su32(bar)), "r"(parity)
                 : "memory");
    return ok;
}

__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, uint32_t limit) {
    for (uint32_t it = 0; it < limit; ++it)
        if (mbar_try(bar, parity)) return true;
    return false;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D (16x8, f32) += A (16x16, f16) * B (16x8, f16)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack_h2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// Four codes of a 32-bit word as two f16 pairs: the low nibble of each half (lo) and the next one (hi).
// EXACT: c - 8 as normal numbers.  Otherwise the subnormals c * 2^-24 and 16 c * 2^-24, one AND each.
template <bool EXACT>
__device__ __forceinline__ void codes_of(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if (EXACT) {
        const uint32_t a = (x & 0x000F000Fu) | 0x64006400u, b = (x & 0x00F000F0u) | 0x64006400u;  // 1024 + c, + 16 c
        const __half2 cl = __hsub2(*reinterpret_cast<const __half2*>(&a), __half2half2(__ushort_as_half(0x6408)));  // 1032
        const __half2 ch = __hfma2(*reinterpret_cast<const __half2*>(&b), __half2half2(__ushort_as_half(0x2C00)),   // 1/16
                                   __half2half2(__ushort_as_half(0xD480)));                                        // -72
        lo = *reinterpret_cast<const uint32_t*>(&cl);
        hi = *reinterpret_cast<const uint32_t*>(&ch);
    } else {
        lo = x & 0x000F000Fu;
        hi = x & 0x00F000F0u;
    }
}

// 2^e, for e within the range of normal floats
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// log2 of a V scale's size, as the choice of a unit for the weights takes it: 2^-25 and less count as 2^-25
__device__ __forceinline__ float log2_scale(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fminf(fmaxf(x, 0x1p-25f), 65504.f)));
    return y;
}

// 2^x of a whole number x within the range of normal floats
__device__ __forceinline__ float pow2_whole(float x) { return __int_as_float(__float_as_int(x + (12582912.f + 127.f)) << 23); }

// x's exponent, cut to a range in which pow2f of it, its negative and small sums are normal
__device__ __forceinline__ int exponent_of(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xFF) - 127;
    return min(max(e, -80), 80);
}

// A unit of work: chunk `chunk` of kv head and row tile `part` of sequence `b`, which has `len` tokens.
struct Cursor {
    uint32_t b, part, chunk, len;
    int32_t row;
};

__device__ __forceinline__ uint32_t kv_head_of(const AttnArgs& a, uint32_t part) { return a.tiles == 1 ? part : part / a.tiles; }

__device__ __forceinline__ uint32_t chunks_of(uint32_t len) { return (len + kKvChunk - 1) / kKvChunk; }

// What a head of a sequence counts in the split of the work: its chunks, and one for its beginning and end
// (operands of q, reductions, results), which cost about as much as a chunk.
__device__ __forceinline__ uint32_t share_of(uint32_t len) { return len ? chunks_of(len) + 1 : 0; }

// Table row and length of batch entry b; row -1: not to be computed.
__device__ __forceinline__ void sequence(const AttnArgs& a, uint32_t b, int32_t* row, uint32_t* len) {
    int32_t r = a.seqs ? a.seqs[b] : (int32_t)b;
    if (r < 0 || (uint32_t)r >= a.rows) r = -1;
    const int32_t l = r < 0 ? 0 : a.lengths[r];
    *row = r;
    *len = l < 0 ? 0u : (uint32_t)min((unsigned long long)l, (unsigned long long)a.width << a.page_shift);
}

__device__ __forceinline__ void advance(const AttnArgs& a, Cursor& c, uint32_t parts) {
    if (++c.chunk < chunks_of(c.len)) return;
    c.chunk = 0;
    if (++c.part < parts) return;
    c.part = 0;
    do {
        if (++c.b >= a.batch) return;
        sequence(a, c.b, &c.row, &c.len);
    } while (c.len == 0);
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8]) {
    if (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        alignas(16) T h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = from_f<T>(v[i]);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
    }
}

}  // namespace

// The work is the list of all (sequence, kv head, row tile, chunk of 64 tokens), in that order, with one
// more place for each head's beginning and end; each warp takes an equal run of it, whatever the lengths, and hands on partial results for the (at most
// two) heads that it shares with its neighbours; k_kv4_join adds those up.  A row tile is 8 NT of the
// kv head's queries * (heads / kv_heads) query rows.  Warps have nothing to do with one another (with
// four of them on one head, joining their sums cost as much as a 1000-token head itself).
//
// A warp feeds itself: per page one bulk copy of the head's codes and parameters into one of its two
// stages while it computes on the other, 16 tokens to a tile, two tiles at a time:
//
//   S^T [token][row] = K codes (A, 16x16) * q (B, 16x8), on mma.sync.  For 16-bit rows: the code
//   0..15 in the low bits of a 16-bit word is the f16 subnormal c * 2^-24, exactly, and in the next
//   four bits 16 c * 2^-24: one AND gives two operand elements, and q is divided by 16 where they are
//   16-fold.
//   Scale and offset stay out of the product: s = scale * (sum q c) + offset * (sum q), in f32.
//   p = 2^(s - m).  The reference m of a row only grows when a score passes it by 8, so that most
//   tiles need no maximum across lanes (one vote); p stays below 2^8.
//   O^T [dim][row] += V codes^T (A) * w (B), w = p * scale, which one movmatrix per 8x8 turns from
//   the accumulator's layout into the operand's.  p * offset is summed apart, in f32 FMAs.
//   w goes in as f16 in units of a power of two of the row's and the group's own, chosen so that the largest
//   w met so far is 16 to 32, and again before one would pass f16's range: a token with a large scale that this row gives no weight to, or the other
//   group's scales, must not take the bits of those that count.  The vote that guards m guards them too.  (A
//   token whose V is nothing but zeros counts as one of scale 2^-25; beside it what lies 2^-50 below is lost.)
//
// With f32 rows (SPLIT) q and w go in as two f16 each, high and remainder, so that products are good
// to 2^-22.  mma.sync aligns products by their operands' exponents, of which a subnormal's is above
// its value, and cuts off what falls below, so f32 rows take the codes as normal numbers, c - 8 (one
// more instruction for two elements, and less to cancel between scale and offset), and sum 32 tokens
// by themselves before the long sum in f32 (4e-6 off without either, 1e-7 with both).  16-bit rows
// need one operand for q (f16 or bf16, it fits f16 after a power of two is taken out).  bf16 rows need one for
// w too: its rounding to f16, half a step 2^-11, is an eighth of the output's half step 2^-8 (at most 1.02
// times the error of f32 sums, with few tokens, whose scale * code cancels against the offset).  In f16 rows it
// would be as large as the output's own (1.7 times), so they take w as two.
//
// Bound: 4.5 bits a value leave two to three instructions a value at full HBM rate, and the loop needs about
// three.  No pipe is at its end, though: 45 to 58 % of the issue slots are used (ALU pipe 35 to 51 %, tensor 17 to
// 24 %), and most of a warp's other cycles go to the fixed latencies of the chain scores - vote - exponential -
// pack - movmatrix - product, which three warps a scheduler do not hide.  256 sequences up to 2048 tokens, 14/2
// heads of 64, f32: 30 us, 1.3 TB/s, a quarter of it at the heads' ends (32 us without their place in the
// split); four up to 131072, 32/8 heads of 128, bf16: 107 us, 4.0 TB/s; 24 up to 5000, 4 queries, f16: 23 us.
// tcgen05 would want the codes widened into shared memory first, which costs more than the products do on
// mma.sync at 8 rows.
// Three CTAs an SM where their 168 registers suffice: left to itself the compiler takes 182 to 189 and two.
template <typename T, int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(kKvWarps * 32, HD * NT <= (SPLIT ? 64 : 128) ? 3 : 2) k_kv4_attn(AttnArgs a) {
    constexpr uint32_t G = HD > 64 ? HD / 64 : 1;         // groups of a row
    constexpr uint32_t W = HD / G / 8;                    // words of a group's codes: 8 (hd 32: 4)
    constexpr uint32_t KW = W / 4;                        // K words a lane takes of a group
    constexpr uint32_t MT = HD / 16;                      // 16-row tiles of O^T
    constexpr uint32_t kRow = HD / 2, kTokenBytes = HD + 8 * G;
    constexpr uint32_t kStageBytes = kKvChunk * kTokenBytes;
    constexpr uint32_t kCols = 8 * NT;
    constexpr bool kTwo = !std::is_same<T, __nv_bfloat16>::value;  // w as two f16 each
    // the operands' units: subnormal codes are 2^-24, and every second one is 16-fold
    constexpr int kExp = SPLIT ? 0 : 24;
    constexpr float kOdd = SPLIT ? 1.f : 0.0625f, kUp = SPLIT ? 1.f : 0x1p24f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kKvWarps][kKvStages];
    __shared__ uint32_t s_scan[kKvWarps], s_before[kKvWarps * 32];

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t group = a.heads / a.kv_heads, rows = a.queries * group, parts = a.kv_heads * a.tiles;

    pdl_launch_dependents();  // the join may take its place where there is room; it waits for this grid's end
    // ---- where this warp's run of units begins --------------------------------------------------
    if (lane < kKvStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(su32(&full[warp][lane])));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    const uint32_t each = (a.batch + 127) / 128, b0 = min(tid * each, a.batch), b1 = min(b0 + each, a.batch);
    uint32_t mine = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        int32_t row;
        uint32_t len;
        sequence(a, b, &row, &len);
        mine += share_of(len) * parts;
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += up;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint32_t before = incl - mine, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kKvWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    s_before[tid] = before;
    const uint32_t runs = gridDim.x * kKvWarps;
    // A head is cut into 257 pieces at most, by the longest that the table can hold: so a table much wider than its
    // sequences makes long runs for few warps (the 256 sequences above: 30 us with 2048 tokens a row, 38 us with
    // 131072, 117 us with 2^20).
    const uint32_t per = max(max(kKvMinRun, (a.most_chunks + 255) / 256), (total + runs - 1) / runs);
    if (blockIdx.x == 0) {  // what the join needs to find the pieces
        uint32_t at = before;
        for (uint32_t b = b0; b < b1; ++b) {
            int32_t row;
            uint32_t len;
            sequence(a, b, &row, &len);
            a.head_ws[b] = at;
            at += share_of(len) * parts;
        }
        if (tid == 0) {
            a.head_ws[a.batch] = total;
            a.head_ws[a.batch + 1] = per;
        }
    }
    __syncthreads();
    const uint32_t run = warp * gridDim.x + blockIdx.x;  // neighbouring runs on different SMs
    const unsigned long long first = (unsigned long long)run * per;
    const uint32_t u0 = (uint32_t)min((unsigned long long)total, first), u1 = min(total, u0 + per);
    if (u0 == u1) return;
    Cursor c{0, 0, 0, 0, -1};
    {
        uint32_t lower = 0;  // threads whose sequences begin at or before u0
#pragma unroll
        for (uint32_t w = 0; w < kKvWarps; ++w) lower += __popc(__ballot_sync(0xffffffffu, s_before[w * 32 + lane] <= u0));
        uint32_t at = s_before[lower - 1];
        c.b = (lower - 1) * each;
        for (;; ++c.b) {
            if (c.b >= a.batch) return;  // (only if the lengths change under the call)
            sequence(a, c.b, &c.row, &c.len);
            const uint32_t n = share_of(c.len) * parts;
            if (u0 < at + n) break;
            at += n;
        }
        // place 0 of a head's share is its beginning, place i chunk i - 1
        c.part = (u0 - at) / share_of(c.len);
        c.chunk = (u0 - at) % share_of(c.len);
    }
    // the chunks among the run's units: a beginning at its end is left to the next run
    uint32_t units = 0;
    {
        Cursor head = c;
        uint32_t left = u1 - u0, place = c.chunk;
        while (left) {
            if (place == 0) {
                --left;
                place = 1;
            }
            const uint32_t take = min(left, share_of(head.len) - place);
            units += take;
            left -= take;
            if (left) {
                head.chunk = chunks_of(head.len) - 1;
                advance(a, head, parts);
                if (head.b >= a.batch) break;
                place = 0;
            }
        }
        c.chunk = c.chunk ? c.chunk - 1 : 0;
    }
    if (units == 0) return;

    // ---- feeding: lane i copies the i-th page of a chunk, or section i of a half page of 128 --------
    const uint32_t limit = g_kv4_spin;
    const uint32_t page_tokens = 1u << a.page_shift, head_bytes = page_tokens * kTokenBytes;
    const uint32_t stage_page = min(page_tokens, kKvChunk), stage_head = stage_page * kTokenBytes;
    uint8_t* ring = smem + warp * (kKvStages * kStageBytes);
    auto page_at = [&](const Cursor& at) -> int32_t {  // -2: nothing for this lane
        const uint32_t token = at.chunk * kKvChunk + (page_tokens > kKvChunk ? 0 : lane << a.page_shift);
        if (page_tokens > kKvChunk ? lane >= 4 : (lane << a.page_shift) >= kKvChunk || token >= at.len) return -2;
        const int32_t p = a.table[(size_t)at.row * a.width + (token >> a.page_shift)];
        return p >= 0 && (uint32_t)p < a.pages ? p : -1;
    };
    uint32_t poison = 0;  // bit s: a page of stage s lies outside the pool
    auto fetch = [&](const Cursor& at, int32_t page, uint32_t s) {
        uint32_t from = 0, onto = lane * head_bytes, bytes = head_bytes;
        if (page_tokens > kKvChunk) {
            const uint32_t half = at.chunk & 1, sec = lane & 1 ? 4 * G : kRow;
            from = (lane >> 1) * (head_bytes / 2) + (lane & 1 ? page_tokens * kRow : 0) + half * kKvChunk * sec;
            onto = (lane >> 1) * (stage_head / 2) + (lane & 1 ? kKvChunk * kRow : 0);
            bytes = kKvChunk * sec;
        }
        const uint32_t mine_bytes = page >= 0 ? bytes : 0;
        const uint32_t all = __reduce_add_sync(0xffffffffu, mine_bytes);
        poison = (poison & ~(1u << s)) | (__any_sync(0xffffffffu, page == -1) ? 1u << s : 0u);
        if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(&full[warp][s])), "r"(all)
                         : "memory");
        __syncwarp();
        if (page >= 0)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             su32(ring + s * kStageBytes + onto)),
                         "l"(a.pool + ((size_t)(uint32_t)page * a.kv_heads + kv_head_of(a, at.part)) * head_bytes + from),
                         "r"(bytes), "r"(su32(&full[warp][s]))
                         : "memory");
    };
    Cursor ahead = c;  // the next unit to be fetched, and this lane's page of it
    int32_t ahead_page = page_at(ahead);
    uint32_t fetched = 0;
    auto fetch_next = [&]() {
        const Cursor now = ahead;
        const int32_t page = ahead_page;
        const uint32_t s = fetched++ % kKvStages;
        if (fetched < units) {  // the table entry after this one is on its way while the copy is set up
            advance(a, ahead, parts);
            ahead_page = page_at(ahead);
        }
        fetch(now, page, s);
    };
    while (fetched < min(units, kKvStages)) fetch_next();

    // ---- computing --------------------------------------------------------------------------------
    const uint32_t g = lane >> 2, t = lane & 3;
    // Token of row i of a 16-token tile: an order in which neither the K rows of a half warp nor the
    // V rows 2t (or 2t + 1) of a warp share a bank.
    auto token_of = [](uint32_t i) { return (i & 8) | ((i & 7) ^ ((i >> 2) & 1)); };
    const uint32_t kt0 = token_of(g), kt1 = kt0 + 8;  // this lane's rows of S^T
    const uint32_t vt[4] = {token_of(2 * t), token_of(2 * t + 1), token_of(2 * t + 8), token_of(2 * t + 9)};
    auto params = [](const uint8_t* at) {  // scale and offset (of c - 8 where that is the operand)
        float2 v = unpack_h2(*reinterpret_cast<const uint32_t*>(at));
        if (SPLIT) v.y = fmaf(8.f, v.x, v.y);
        return v;
    };

    uint32_t qf[NT][G * KW * 2][2], ql[SPLIT ? NT : 1][SPLIT ? G * KW * 2 : 1][2];
    float kfac[NT][2], qsum[NT][2][G];
    int32_t last[NT][2];  // the last token a column sees
    // m: a row's reference, lu: log2 of the unit of its weights in each group, a whole number
    float m[NT][2], l[NT][2], o[NT][MT][4], om[NT][2][G], lu[NT][2][G];

    uint32_t begun = 0;  // the unit of the run with which the present head began
    bool gave_up = false;
    for (uint32_t i = 0; i < units; ++i) {
        if (i == 0 || c.chunk == 0) {
            // ---- a new head: its queries as operands, columns 8 n + g --------------------------------
            begun = i;
            const uint32_t kvh = kv_head_of(a, c.part), tile = c.part - kvh * a.tiles;
            float qs[NT][G];
            int qe[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t r = (tile * NT + n) * 8 + g;
                const T* qp = nullptr;
                if (r < rows)
                    qp = static_cast<const T*>(a.q) + (long long)c.b * a.q_seq + (long long)(r / group) * a.q_query +
                         (long long)(kvh * group + r % group) * a.q_head;
                float x[G * KW][8], top = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < G * KW; ++w) {  // lane t: words KW t .. of each group
                    const T* src = qp + (w / KW) * 64 + (KW * t + w % KW) * 8;
                    alignas(16) T raw[8];
                    if (qp && a.vec) {
#pragma unroll
                        for (uint32_t e = 0; e < sizeof(T) / 2; ++e)
                            reinterpret_cast<uint4*>(raw)[e] = __ldg(reinterpret_cast<const uint4*>(src) + e);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) raw[e] = qp ? src[e] : from_f<T>(0.f);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[w][e] = to_f(raw[e]);
                        top = fmaxf(top, fabsf(x[w][e]));
                    }
                }
#pragma unroll
                for (uint32_t gr = 0; gr < G; ++gr) {
                    float sum = 0.f;
#pragma unroll
                    for (uint32_t w = 0; w < KW; ++w)
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum += x[gr * KW + w][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    qs[n][gr] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                qe[n] = exponent_of(top);
                const float up = pow2f(13 - qe[n]);  // the row's largest at 2^13
#pragma unroll
                for (uint32_t w = 0; w < G * KW; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int odd = 0; odd < 2; ++odd) {
                            const float f = odd ? up * kOdd : up;
                            const float v0 = x[w][2 * h + odd] * f, v1 = x[w][2 * h + odd + 4] * f;
                            qf[n][2 * w + h][odd] = pack_h2(v0, v1);
                            if (SPLIT) {
                                const float2 back = unpack_h2(qf[n][2 * w + h][odd]);
                                ql[n][2 * w + h][odd] = pack_h2(v0 - back.x, v1 - back.y);
                            }
                        }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // this lane's columns 2t + j: their lanes hold them as g
                    const int src = (2 * t + j) * 4;
                    kfac[n][j] = pow2f(kExp + __shfl_sync(0xffffffffu, qe[n], src) - 13) * a.scale_log2;
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr) qsum[n][j][gr] = __shfl_sync(0xffffffffu, qs[n][gr], src) * a.scale_log2;
                    const uint32_t r = (tile * NT + n) * 8 + 2 * t + j;
                    last[n][j] = (int32_t)c.len - (int32_t)a.queries + (int32_t)min(r / group, a.queries - 1);
                    m[n][j] = kKvLow;
                    l[n][j] = 0.f;
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr) om[n][j][gr] = lu[n][j][gr] = 0.f;
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t d = 0; d < MT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][d][e] = 0.f;
        }

        const uint32_t s = i % kKvStages;
        // A wait that gives up: the error is raised, nothing more is computed or fetched.
        if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][s], (i / kKvStages) & 1, limit))) {
            gave_up = true;
            break;
        }
        const uint8_t* stage = ring + s * kStageBytes;
        const uint32_t chunk0 = c.chunk * kKvChunk;
        const bool edge = chunk0 + kKvChunk + a.queries > c.len + 1;  // some column may not see it all
        if (poison >> s & 1) {  // a page number outside the pool: the sequence's rows become NaN
#pragma unroll
            for (int n = 0; n < NT; ++n) l[n][0] = l[n][1] = __int_as_float(0x7fffffff);
        }
        // Two tiles of 16 tokens from `tok` of the chunk on, each within one page: twice the independent
        // work between the votes and the long chains of products.
        auto tiles32 = [&](uint32_t tok, auto is_edge) {
            constexpr bool kEdge = decltype(is_edge)::value;
            const uint8_t* vc[2];
            float sc[2][NT][4];
            float2 v0[2][G], v1[2][G];  // V parameters of this lane's tokens
            // what a column does not see, and what lies behind the sequence, counts for nothing whatever it holds
            auto hidden = [&](int p, int n, int e) {
                return kEdge && (int32_t)(chunk0 + tok + 16 * p + (e < 2 ? kt0 : kt1)) > last[n][e & 1];
            };
            float vtop[G] = {};  // the largest scale of this lane's tokens
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t at = tok + 16 * p, in_page = at & (stage_page - 1);
                const uint8_t* base = stage + (at >> a.page_shift) * stage_head;
                const uint8_t* kc = base + in_page * kRow;
                const uint8_t* kp = base + stage_page * kRow + in_page * (4 * G);
                const uint8_t* vp = kp + stage_head / 2;
                vc[p] = kc + stage_head / 2;
                // S^T
#pragma unroll
                for (uint32_t gr = 0; gr < G; ++gr) {
                    uint32_t w0[KW], w1[KW];
                    if (KW == 2) {
                        const uint2 r0 = *reinterpret_cast<const uint2*>(kc + kt0 * kRow + gr * 32 + t * 8);
                        const uint2 r1 = *reinterpret_cast<const uint2*>(kc + kt1 * kRow + gr * 32 + t * 8);
                        w0[0] = r0.x, w0[KW - 1] = r0.y, w1[0] = r1.x, w1[KW - 1] = r1.y;
                    } else {
                        w0[0] = *reinterpret_cast<const uint32_t*>(kc + kt0 * kRow + t * 4);
                        w1[0] = *reinterpret_cast<const uint32_t*>(kc + kt1 * kRow + t * 4);
                    }
                    float acc[KW][NT][4];
#pragma unroll
                    for (uint32_t w = 0; w < KW; ++w) {
                        uint32_t af[2][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            codes_of<SPLIT>(h ? w0[w] >> 8 : w0[w], af[h][0], af[h][2]);
                            codes_of<SPLIT>(h ? w1[w] >> 8 : w1[w], af[h][1], af[h][3]);
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint32_t f = 2 * (gr * KW + w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[w][n][e] = 0.f;
                            if (SPLIT) {  // the small remainders first, before there is a sum to cut them to
                                mma16816(acc[w][n], af[0], ql[n][f][0], ql[n][f][1]);
                                mma16816(acc[w][n], af[1], ql[n][f + 1][0], ql[n][f + 1][1]);
                            }
                            mma16816(acc[w][n], af[0], qf[n][f][0], qf[n][f][1]);
                            mma16816(acc[w][n], af[1], qf[n][f + 1][0], qf[n][f + 1][1]);
                        }
                    }
                    const float2 p0 = params(kp + (kt0 * G + gr) * 4), p1 = params(kp + (kt1 * G + gr) * 4);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 pp = e < 2 ? p0 : p1;
                            const float sum = KW == 2 ? acc[0][n][e] + acc[KW - 1][n][e] : acc[0][n][e];
                            const float off = pp.y * qsum[n][e & 1][gr];
                            sc[p][n][e] = fmaf(sum * kfac[n][e & 1], pp.x, gr == 0 ? off : off + sc[p][n][e]);
                        }
                    v0[p][gr] = params(vp + (kt0 * G + gr) * 4);
                    v1[p][gr] = params(vp + (kt1 * G + gr) * 4);
                }
                if (kEdge) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (hidden(p, n, e)) sc[p][n][e] = -INFINITY;
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr) {
                        if (chunk0 + at + kt0 >= c.len) v0[p][gr] = make_float2(0.f, 0.f);
                        if (chunk0 + at + kt1 >= c.len) v1[p][gr] = make_float2(0.f, 0.f);
                    }
                }
#pragma unroll
                for (uint32_t gr = 0; gr < G; ++gr) vtop[gr] = fmaxf(vtop[gr], fmaxf(fabsf(v0[p][gr].x), fabsf(v1[p][gr].x)));
            }
            // a weight scale * 2^(s - m + lu) has to stay below 2^16, and s - m below 8
            float room[G];
#pragma unroll
            for (uint32_t gr = 0; gr < G; ++gr) room[gr] = 15.5f - log2_scale(vtop[gr]);
            bool over = false;
            float tops[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    tops[n][j] = fmaxf(fmaxf(sc[0][n][j], sc[0][n][2 + j]), fmaxf(sc[1][n][j], sc[1][n][2 + j]));
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr)
                        over = over || tops[n][j] - m[n][j] > fminf(8.f, room[gr] - lu[n][j][gr]);
                }
            if (__any_sync(0xffffffffu, over)) {
                // New references: the maxima of the rows that are past theirs (themselves, unrounded: the weight of a
                // token that has it all is then 1, and its scale loses nothing in f16).  New units: the largest weight
                // so far comes to 16 to 32 (what the unit says of the earlier ones, less what the reference's move
                // takes off, or this tile's).  A move of 8 and more costs that estimate less than 1 in rounding.
                float lv[2][2][G];
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr) {
                        lv[p][0][gr] = log2_scale(fabsf(v0[p][gr].x));
                        lv[p][1][gr] = log2_scale(fabsf(v1[p][gr].x));
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[G][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = tops[n][j], wide[G];
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        top = top - m[n][j] > 8.f ? top : m[n][j];
                        const float moved = top - m[n][j], fm = ex2(-moved);
                        m[n][j] = top;
                        l[n][j] *= fm;
#pragma unroll
                        for (uint32_t gr = 0; gr < G; ++gr) {
                            wide[gr] = -INFINITY;
#pragma unroll
                            for (int p = 0; p < 2; ++p)
                                wide[gr] = fmaxf(wide[gr], fmaxf(sc[p][n][j] - top + lv[p][0][gr], sc[p][n][2 + j] - top + lv[p][1][gr]));
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) wide[gr] = fmaxf(wide[gr], __shfl_xor_sync(0xffffffffu, wide[gr], x));
                            const float unit = 4.f - floorf(fmaxf(wide[gr], 4.f - lu[n][j][gr] - moved));
                            f[gr][j] = fm * pow2_whole(unit - lu[n][j][gr]);
                            lu[n][j][gr] = unit;
                            om[n][j][gr] *= fm;
                        }
                    }
#pragma unroll
                    for (uint32_t d = 0; d < MT; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][d][e] *= f[G == 1 ? 0 : d / 4][e & 1];
                }
            }
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[p][n][e] = ex2(sc[p][n][e] - m[n][e & 1]);
                        l[n][e & 1] += sc[p][n][e];
                    }

            // O^T
#pragma unroll
            for (uint32_t gr = 0; gr < G; ++gr) {
                uint32_t wb[2][NT][2], wl[2][NT][2];
                float unit[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) unit[n][j] = pow2_whole(lu[n][j][gr]);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x[e] = hidden(p, n, e) ? 0.f : sc[p][n][e] * ((e < 2 ? v0 : v1)[p][gr].x * unit[n][e & 1]);
                        const uint32_t h0 = pack_h2(x[0], x[1]), h1 = pack_h2(x[2], x[3]);
                        wb[p][n][0] = transpose8x8(h0);
                        wb[p][n][1] = transpose8x8(h1);
                        if (kTwo) {
                            const float2 r0 = unpack_h2(h0), r1 = unpack_h2(h1);
                            wl[p][n][0] = transpose8x8(pack_h2(x[0] - r0.x, x[1] - r0.y));
                            wl[p][n][1] = transpose8x8(pack_h2(x[2] - r1.x, x[3] - r1.y));
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if (!hidden(p, n, j)) om[n][j][gr] = fmaf(sc[p][n][j], v0[p][gr].y, om[n][j][gr]);
                            if (!hidden(p, n, 2 + j)) om[n][j][gr] = fmaf(sc[p][n][2 + j], v1[p][gr].y, om[n][j][gr]);
                        }
                    }
                }
                // lane g: word g of the group's row (hd 32: half a word), of this lane's four tokens of each tile
                uint32_t w[2][4];
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[p][j] = *reinterpret_cast<const uint32_t*>(vc[p] + vt[j] * kRow + gr * 32 + (W == 8 ? g : g >> 1) * 4);
#pragma unroll
                for (uint32_t hw = 0; hw < W / 4; ++hw) {  // 16-bit halves of the words: dims 4 hw ..
                    const uint32_t sel = W == 8 ? (hw ? 0x7632u : 0x5410u) : (g & 1 ? 0x7632u : 0x5410u);
                    uint32_t a0[2], a1[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        a0[p] = __byte_perm(w[p][0], w[p][1], sel);
                        a1[p] = __byte_perm(w[p][2], w[p][3], sel);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t af[2][4];
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            codes_of<SPLIT>(h ? a0[p] >> 8 : a0[p], af[p][0], af[p][1]);
                            codes_of<SPLIT>(h ? a1[p] >> 8 : a1[p], af[p][2], af[p][3]);
                        }
                        const uint32_t d = gr * 4 + 2 * hw + h;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (SPLIT) {  // 32 tokens' sum by itself: the long one is rounded, not cut, in f32
                                float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int p = 0; p < 2; ++p) mma16816(add, af[p], wl[p][n][0], wl[p][n][1]);
#pragma unroll
                                for (int p = 0; p < 2; ++p) mma16816(add, af[p], wb[p][n][0], wb[p][n][1]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[n][d][e] += add[e];
                            } else {
                                if (kTwo) {
#pragma unroll
                                    for (int p = 0; p < 2; ++p) mma16816(o[n][d], af[p], wl[p][n][0], wl[p][n][1]);
                                }
#pragma unroll
                                for (int p = 0; p < 2; ++p) mma16816(o[n][d], af[p], wb[p][n][0], wb[p][n][1]);
                            }
                        }
                    }
                }
            }
        };
        if (!edge) {
#pragma unroll 1
            for (uint32_t tok = 0; tok < kKvChunk; tok += 32) tiles32(tok, std::false_type{});
        } else {
#pragma unroll 1
            for (uint32_t tok = 0; tok < kKvChunk && chunk0 + tok < c.len; tok += 32) tiles32(tok, std::true_type{});
        }
        __syncwarp();  // every lane has read the stage
        if (fetched < units) fetch_next();

        const bool head_done = c.chunk + 1 == chunks_of(c.len);
        if (head_done || i + 1 == units) {
            // ---- the head's result, or this run's part of it --------------------------------------------
            const uint32_t kvh = kv_head_of(a, c.part), tile = c.part - kvh * a.tiles;
            const bool whole = head_done && i - begun == c.chunk;
            // the run's first head goes to slot 0 of its two, one that began later to slot 1
            float* part = a.part + (size_t)(2 * run + (begun ? 1 : 0)) * kCols * (HD + 4);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float lt = l[n][j], mt[G], back[G];
#pragma unroll
                    for (uint32_t gr = 0; gr < G; ++gr) {
                        mt[gr] = om[n][j][gr];
                        back[gr] = kUp * pow2_whole(-lu[n][j][gr]);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        lt += __shfl_xor_sync(0xffffffffu, lt, x);
#pragma unroll
                        for (uint32_t gr = 0; gr < G; ++gr) mt[gr] += __shfl_xor_sync(0xffffffffu, mt[gr], x);
                    }
                    const uint32_t col = n * 8 + 2 * t + j, r = tile * kCols + col;
                    if (r >= rows) continue;
                    const float inv = whole ? (lt == 0.f ? 0.f : 1.f / lt) : 1.f;
                    T* dst = static_cast<T*>(a.out) +
                             (((size_t)c.b * a.queries + r / group) * a.heads + kvh * group + r % group) * HD;
                    float* pd = part + col * (HD + 4);
                    // tile d: dims 2 (d % 4) and + 1 of this lane's run of 8 (hd 32: of 4)
                    if (HD > 32) {
#pragma unroll
                        for (uint32_t gr = 0; gr < G; ++gr) {
                            float v[8];
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                v[2 * d] = fmaf(o[n][gr * 4 + d][j], back[gr], mt[gr]) * inv;
                                v[2 * d + 1] = fmaf(o[n][gr * 4 + d][2 + j], back[gr] * kOdd, mt[gr]) * inv;
                            }
                            if (whole)
                                store8(dst + gr * 64 + g * 8, v);
                            else
                                store8(pd + gr * 64 + g * 8, v);
                        }
                    } else {
#pragma unroll
                        for (uint32_t d = 0; d < MT; ++d) {
                            const float x0 = fmaf(o[n][d][j], back[0], mt[0]) * inv, x1 = fmaf(o[n][d][2 + j], back[0] * kOdd, mt[0]) * inv;
                            if (whole) {
                                dst[g * 4 + 2 * d] = from_f<T>(x0);
                                dst[g * 4 + 2 * d + 1] = from_f<T>(x1);
                            } else {
                                pd[g * 4 + 2 * d] = x0;
                                pd[g * 4 + 2 * d + 1] = x1;
                            }
                        }
                    }
                    if (!whole && g == 0) {
                        pd[HD] = m[n][j];
                        pd[HD + 1] = lt;
                    }
                }
        }
        advance(a, c, parts);
    }
    if (gave_up) {
        if (lane == 0) atomicMax(&g_kv4_err, 1u);
        // no copy may still be landing when the CTA releases its shared memory
        for (uint32_t i = fetched > kKvStages ? fetched - kKvStages : 0; i < fetched; ++i)
            mbar_wait(&full[warp][i % kKvStages], (i / kKvStages) & 1, kKvSpin);
    }
}

// Joins the partial results of the heads that more than one run shared, in the order of the runs,
// and writes zeros for sequences of length 0.  A block per (sequence, kv head, row tile) and COLS of
// its rows; a thread has 4 dims of one row, the rest of the block shares the pieces.
template <typename T, int HD, int NT, int COLS>
__global__ void __launch_bounds__(256) k_kv4_join(AttnArgs a) {
    constexpr uint32_t kCols = 8 * NT, kLanes = HD / 4, kSplit = 256 / kLanes / COLS;
    __shared__ float4 s_acc[kSplit][COLS * kLanes];
    __shared__ float s_l[kSplit][COLS], s_top[kSplit][COLS];
    pdl_wait();
    const uint32_t group = a.heads / a.kv_heads, rows = a.queries * group, tid = threadIdx.x;
    const uint32_t parts = a.kv_heads * a.tiles, part = blockIdx.x % parts, b = blockIdx.x / parts;
    int32_t row;
    uint32_t len;
    sequence(a, b, &row, &len);
    if (row < 0) return;
    const uint32_t per = a.head_ws[a.batch + 1], n = share_of(len);
    const uint32_t u0 = a.head_ws[b] + part * n;  // the head's beginning; its chunks follow
    const uint32_t c0 = (u0 + 1) / per, c1 = len ? (u0 + n - 1) / per : c0 + 1;
    if (c0 == c1) return;  // one run had it all
    const uint32_t kvh = part / a.tiles, d4 = tid % kLanes, local = tid / kLanes % COLS, share = tid / kLanes / COLS;
    const uint32_t col = blockIdx.y * COLS + local, r = part % a.tiles * kCols + col;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float ls = 0.f;
    if (len) {
        // run c's piece is the first of the run (slot 0) or, only for c0, comes behind another head's (slot 1)
        auto piece = [&](uint32_t c) {
            return a.part + ((size_t)(2 * c + (u0 > c * per ? 1 : 0)) * kCols + col) * (HD + 4);
        };
        float top = kKvLow;
        if (r < rows) {
#pragma unroll 4
            for (uint32_t c = c0 + share; c <= c1; c += kSplit) top = fmaxf(top, piece(c)[HD]);
        }
        if (d4 == 0) s_top[share][local] = top;
        __syncthreads();
#pragma unroll
        for (uint32_t p = 0; p < kSplit; ++p) top = fmaxf(top, s_top[p][local]);
        if (r < rows) {
#pragma unroll 4
            for (uint32_t c = c0 + share; c <= c1; c += kSplit) {
                const float* p = piece(c);
                const float f = ex2(p[HD] - top);
                const float4 v = reinterpret_cast<const float4*>(p)[d4];
                sum = make_float4(fmaf(f, v.x, sum.x), fmaf(f, v.y, sum.y), fmaf(f, v.z, sum.z), fmaf(f, v.w, sum.w));
                ls = fmaf(f, p[HD + 1], ls);
            }
        }
        s_acc[share][tid % (COLS * kLanes)] = sum;
        if (d4 == 0) s_l[share][local] = ls;
        __syncthreads();
    }
    if (share || r >= rows) return;
#pragma unroll 4
    for (uint32_t p = 1; p < kSplit && len; ++p) {
        const float4 v = s_acc[p][tid];
        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
        ls += s_l[p][local];
    }
    const float inv = ls == 0.f ? 0.f : 1.f / ls;
    T* dst = static_cast<T*>(a.out) + (((size_t)b * a.queries + r / group) * a.heads + kvh * group + r % group) * HD + d4 * 4;
    dst[0] = from_f<T>(sum.x * inv);
    dst[1] = from_f<T>(sum.y * inv);
    dst[2] = from_f<T>(sum.z * inv);
    dst[3] = from_f<T>(sum.w * inv);
}

// ---- launches -----------------------------------------------------------------------------------

namespace {

constexpr int kKvDevices = 64, kKvMaxPerSm = 4;
constexpr uint32_t kKvMaxRuns = 148 * kKvMaxPerSm * kKvWarps;  // of a call: the workspace has slots for them

uint32_t log2_of(uint32_t v) {
    uint32_t s = 0;
    while ((1u << s) < v) ++s;
    return s;
}

template <typename T, int HD, int NT, bool SPLIT>
cudaError_t launch_attn4(AttnArgs a, uint64_t most_units, cudaStream_t st) {
    constexpr size_t smem = kKvWarps * kKvStages * kKvChunk * (HD + 8 * (HD > 64 ? HD / 64 : 1));
    static std::atomic<int> known[kKvDevices];  // per device: CTAs an SM holds, over which the units are split
    int dev = 0, per_sm = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < kKvDevices) per_sm = known[dev].load(std::memory_order_acquire);
    if (per_sm == 0) {
        e = cudaFuncSetAttribute(k_kv4_attn<T, HD, NT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k_kv4_attn<T, HD, NT, SPLIT>, kKvWarps * 32, smem);
        if (e != cudaSuccess) return e;
        per_sm = per_sm < 1 ? 1 : (per_sm > kKvMaxPerSm ? kKvMaxPerSm : per_sm);
        if (dev < kKvDevices) known[dev].store(per_sm, std::memory_order_release);
    }
    const uint32_t grid = (uint32_t)(most_units < 148ull * per_sm ? most_units : 148ull * per_sm);
    k_kv4_attn<T, HD, NT, SPLIT><<<grid, kKvWarps * 32, smem, st>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    // few heads: a block per row, as their pieces are many; else blocks of 8 rows (which hd 128 fills)
    const uint32_t heads = a.batch * a.kv_heads * a.tiles;
    const bool few = heads <= 148;
    cfg.gridDim = dim3(heads, few ? 8 * NT : NT);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return few ? cudaLaunchKernelEx(&cfg, k_kv4_join<T, HD, NT, 1>, a) : cudaLaunchKernelEx(&cfg, k_kv4_join<T, HD, NT, 8>, a);
}

template <typename T, bool SPLIT>
cudaError_t pick_attn4(const AttnArgs& a, uint32_t hd, uint32_t nt, uint64_t units, cudaStream_t st) {
    if (hd == 32) return nt == 1 ? launch_attn4<T, 32, 1, SPLIT>(a, units, st) : launch_attn4<T, 32, 2, SPLIT>(a, units, st);
    if (hd == 64) return nt == 1 ? launch_attn4<T, 64, 1, SPLIT>(a, units, st) : launch_attn4<T, 64, 2, SPLIT>(a, units, st);
    return nt == 1 ? launch_attn4<T, 128, 1, SPLIT>(a, units, st) : launch_attn4<T, 128, 2, SPLIT>(a, units, st);
}

enx_status check_cache(const enx_kv4_dims* d, const std::string& w) {
    if (!d) return fail(ENX_ERR_INVALID, w + ": null dims");
    if (d->dtype > ENX_BF16) return fail(ENX_ERR_INVALID, w + ": dtype must be ENX_F32, ENX_F16 or ENX_BF16");
    if (d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128)
        return fail(ENX_ERR_INVALID, w + ": head_dim must be 32, 64 or 128");
    if (d->page_tokens != 16 && d->page_tokens != 32 && d->page_tokens != 64 && d->page_tokens != 128)
        return fail(ENX_ERR_INVALID, w + ": page_tokens must be 16, 32, 64 or 128");
    if (d->kv_heads == 0 || d->kv_heads > 1024) return fail(ENX_ERR_RANGE, w + ": kv_heads must be 1 to 1024");
    if (d->rows == 0 || d->width == 0 || d->pages == 0 || d->pages > (1u << 28))
        return fail(ENX_ERR_RANGE, w + ": rows and width must be positive and pages 1 to 2^28");
    if ((uint64_t)d->width * d->page_tokens > 0x7fffffffull)
        return fail(ENX_ERR_RANGE, w + ": a row may hold at most 2^31 - 1 tokens");
    return ENX_OK;
}

}  // namespace

cudaError_t kv4_set_spin(uint32_t spins) {
    const uint32_t v = spins ? spins : kKvSpin;
    return cudaMemcpyToSymbol(g_kv4_spin, &v, sizeof(v));
}

cudaError_t kv4_take_error(uint32_t* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_kv4_err, sizeof(*code));
    const uint32_t zero = 0;
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_kv4_err, &zero, sizeof(zero));
    return e;
}

}  // namespace enx

using namespace enx;

static enx_status kv4_write(const std::string& w, const void* k, const void* v, const int64_t* strides, uint32_t tokens,
                            uint8_t* pool, const int32_t* table, const int32_t* lengths, const int32_t* seqs,
                            const int32_t* positions, void* k_out, void* v_out, const enx_kv4_dims* d, void* stream) {
    ENX_TRY(check_cache(d, w));
    if (tokens == 0) return ENX_OK;
    if (!k || !v || !strides || !pool || !table || !seqs || !positions) return fail(ENX_ERR_INVALID, w + ": null pointer");
    if (reinterpret_cast<uintptr_t>(pool) % 16) return fail(ENX_ERR_INVALID, w + ": the pool must be 16-byte aligned");
    WriteArgs a{k, v, k_out, v_out, strides[0], strides[1], strides[2], strides[3], pool, table, seqs, positions, lengths, tokens,
                d->rows, d->width, d->pages, log2_of(d->page_tokens), d->kv_heads, d->head_dim, log2_of(d->head_dim / 8), 0};
    const size_t size = d->dtype == ENX_F32 ? 4 : 2;
    uintptr_t any = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_out) |
                    reinterpret_cast<uintptr_t>(v_out);
    for (int i = 0; i < 4; ++i) any |= (uintptr_t)strides[i] * size;
    a.vec = any % 16 == 0;
    const uint64_t threads = (uint64_t)tokens * d->kv_heads * (d->head_dim / 8), blocks = (threads + 255) / 256;
    const uint32_t grid = (uint32_t)blocks;
    if (blocks * 256 > 0xffffffffull) return fail(ENX_ERR_RANGE, w + ": too many tokens for one call");
    if (d->dtype == ENX_F32)
        k_kv4_write<float><<<grid, 256, 0, as_stream(stream)>>>(a);
    else if (d->dtype == ENX_F16)
        k_kv4_write<__half><<<grid, 256, 0, as_stream(stream)>>>(a);
    else
        k_kv4_write<__nv_bfloat16><<<grid, 256, 0, as_stream(stream)>>>(a);
    ENX_CUDA(cudaGetLastError());
    return ENX_OK;
}

extern "C" enx_status enx_kv4_write(const void* k, const void* v, const int64_t* strides, uint32_t tokens,
                                    uint8_t* pool, const int32_t* table, const int32_t* seqs, const int32_t* positions,
                                    void* k_out, void* v_out, const enx_kv4_dims* d, void* stream) {
    return kv4_write("enx_kv4_write", k, v, strides, tokens, pool, table, nullptr, seqs, positions, k_out, v_out, d, stream);
}

extern "C" enx_status enx_kv4_write_held(const void* k, const void* v, const int64_t* strides, uint32_t tokens,
                                         uint8_t* pool, const int32_t* table, const int32_t* lengths, const int32_t* seqs,
                                         const int32_t* positions, void* k_out, void* v_out, const enx_kv4_dims* d,
                                         void* stream) {
    if (tokens && !lengths) return fail(ENX_ERR_INVALID, "enx_kv4_write_held: null pointer");
    return kv4_write("enx_kv4_write_held", k, v, strides, tokens, pool, table, lengths, seqs, positions, k_out, v_out, d, stream);
}

extern "C" size_t enx_attn_kv4_workspace_bytes(uint32_t batch, uint32_t head_dim) {
    return ((size_t)batch + 2 + 63) / 64 * 256 + (size_t)2 * kKvMaxRuns * 16 * (head_dim + 4) * sizeof(float);
}

extern "C" enx_status enx_attn_kv4(const void* q, const int64_t* strides, const uint8_t* pool, const int32_t* table,
                                   const int32_t* lengths, const int32_t* seqs, void* out, uint32_t batch,
                                   uint32_t queries, uint32_t heads, float scale, const enx_kv4_dims* d,
                                   void* workspace, void* stream) {
    ENX_TRY(check_cache(d, "enx_attn_kv4"));
    if (batch == 0 || queries == 0) return ENX_OK;
    if (!q || !strides || !pool || !table || !lengths || !out || !workspace)
        return fail(ENX_ERR_INVALID, "enx_attn_kv4: null pointer");
    if (reinterpret_cast<uintptr_t>(pool) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(ENX_ERR_INVALID, "enx_attn_kv4: pool and workspace must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(out) % 16) return fail(ENX_ERR_INVALID, "enx_attn_kv4: out must be 16-byte aligned");
    if (heads == 0 || heads % d->kv_heads) return fail(ENX_ERR_INVALID, "enx_attn_kv4: heads must be a multiple of kv_heads");
    if (!seqs && batch > d->rows) return fail(ENX_ERR_RANGE, "enx_attn_kv4: more sequences than table rows");
    const uint64_t rows = (uint64_t)queries * (heads / d->kv_heads);
    if (rows > 65536 || (uint64_t)batch * queries * heads > 0x7fffffffull)
        return fail(ENX_ERR_RANGE, "enx_attn_kv4: too many query rows for one call");
    const uint32_t nt = rows <= 8 ? 1 : 2, tiles = (uint32_t)((rows + 8 * nt - 1) / (8 * nt));
    const uint64_t chunks = ((uint64_t)d->width * d->page_tokens + kKvChunk - 1) / kKvChunk + 1;  // and a head's beginning
    if ((uint64_t)batch * d->kv_heads * tiles > 0x7fffffffull / chunks)
        return fail(ENX_ERR_RANGE, "enx_attn_kv4: batch x table width is too large for one call");
    const uint64_t units = (uint64_t)batch * d->kv_heads * tiles * chunks;
    if (!(scale > 0.f)) return fail(ENX_ERR_INVALID, "enx_attn_kv4: scale must be positive");
    AttnArgs a{};
    a.q = q;
    a.q_seq = strides[0];
    a.q_query = strides[1];
    a.q_head = strides[2];
    a.pool = pool;
    a.table = table;
    a.lengths = lengths;
    a.seqs = seqs;
    a.out = out;
    a.head_ws = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ((size_t)batch + 2 + 63) / 64 * 256);
    a.batch = batch;
    a.queries = queries;
    a.heads = heads;
    a.kv_heads = d->kv_heads;
    a.rows = d->rows;
    a.width = d->width;
    a.pages = d->pages;
    a.page_shift = log2_of(d->page_tokens);
    a.tiles = tiles;
    a.most_chunks = (uint32_t)chunks;
    uintptr_t any = reinterpret_cast<uintptr_t>(q);
    for (int i = 0; i < 3; ++i) any |= (uintptr_t)strides[i] * (d->dtype == ENX_F32 ? 4 : 2);
    a.vec = any % 16 == 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    if (d->dtype == ENX_F32)
        ENX_CUDA((pick_attn4<float, true>(a, d->head_dim, nt, units, as_stream(stream))));
    else if (d->dtype == ENX_F16)
        ENX_CUDA((pick_attn4<__half, false>(a, d->head_dim, nt, units, as_stream(stream))));
    else
        ENX_CUDA((pick_attn4<__nv_bfloat16, false>(a, d->head_dim, nt, units, as_stream(stream))));
    return ENX_OK;
}
