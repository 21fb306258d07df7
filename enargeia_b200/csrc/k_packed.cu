// Causal attention over whole prompts packed one behind another, with grouped heads, in f16 or bf16, on
// the 5th-generation tensor cores (tcgen05, TMEM accumulators).
//
// out[i] = sum_j softmax_j(scale * q[i].k[j]) v[j] over the keys j <= i of token i's own prompt.
//
// An item of work is 256 consecutive queries of one prompt and head, as two tiles of 128 rows that take
// turns: while one warpgroup turns the first tile's scores into weights, the tensor cores multiply for
// the second.  Keys go by in tiles of 128, counted from the prompt's start like the rows, so that of
// each row tile only the last key tile needs a mask.  Per key tile and row tile:
//
//   S (TMEM, f32) = Q K^T           kind::f16, M = N = 128, both operands K-major from shared memory
//   p = 2^(scale' (s - m)), to TMEM over S, in 16 bits
//   O (TMEM, f32) += P V            A from TMEM, V MN-major from shared memory as it lies in memory
//
// m, a row's reference, starts as the first key tile's maximum and moves only when a score passes it by
// more than 2^8 in its weight; then the warpgroup rescales its rows of O in TMEM, which is rare.  Sums
// are f32.  Weights are rounded to the inputs' 16 bits for the product, as the output is.
//
// Bound: one exponential per score against 4 hd multiply-adds.  At 16 a clock and SM, 128 x 128 scores
// are 1024 clocks, their products 512 at hd 64 and 1024 at hd 128; so at hd 128 some exponentials are
// taken on the FMA pipe instead (2^x = 2^n 2^f, a cubic in f).
//
// Measured: 16 prompts up to 2048 tokens, 14/2 heads of 64, 115 us (414 TFLOP/s); three up to 12001, 32/8 heads of
// 128, 1440 us (1040 TFLOP/s) in passes one behind another, where the card is at its 1000 W and runs at 1640 MHz,
// and 1274 us (1174 TFLOP/s) alone; one of 16384, 16/2 heads, alone, 741 and 1239 TFLOP/s at hd 64 and 128.
//
// One CTA per SM works through items, the next one's loads and first products under the present one's
// last weights and output.  Items are in descending order of their key tiles, over all prompts and
// heads, and dealt out to and fro (CTA c takes items c, 2G - 1 - c, 2G + c, ..), which keeps the CTAs'
// shares even without a counter.
//
// Warp roles, synchronised by mbarriers with bounded waits:
//   warps 0, 3      issue the products: hd 64, scores and outputs, hd 128, row tile 0 and 1 (and warp 0
//                   owns TMEM)
//   warp 1          lane 0 loads Q, K and V tiles by TMA (128-byte swizzle; 64-element halves of a row)
//   warp 2          finds the items
//   warps 4-7, 8-11 softmax of row tile 0 and 1 (thread = row)
//   warps 12-15     output of both row tiles; and the V tiles that some row sees only in part (below)
//
// A weight of zero times a V element that is not finite would be NaN.  The last two key tiles of an item
// are the only ones that hold keys which some row does not see, so in those the output warps replace
// such elements by zeros before the product, and where there were any, each row adds those that it does
// see to its output.

#include <cuda.h>
#include <cuda_bf16.h>

#include <atomic>

#include "enx_internal.cuh"
#include "k_packed.cuh"

namespace enx {

namespace {

constexpr uint32_t kPkSpin = 1u << 24;  // default limit of a wait, and the limit of the drain waits
__device__ uint32_t g_packed_spin = kPkSpin;
__device__ uint32_t g_packed_err = 0;

constexpr uint32_t kPkRows = 128;           // rows of a tile, keys of a tile
constexpr uint32_t kPkThreads = 512;
constexpr uint32_t kPkItems = 4;             // items between the warp that finds them and the others
constexpr uint32_t kPkClean = 4;             // barriers of partly seen V tiles: more than a ring holds
constexpr uint32_t kPkFoul = 2;              // flags of items whose partly seen V tiles were not all finite (below)
constexpr uint32_t kPkTileBytes = 128 * 128;  // 128 rows of 64 16-bit elements
constexpr int kPkRegs = 128, kPkRegsSoftmax = 192, kPkRegsOut = 88, kPkRegsRest = 40;
static_assert(2 * kPkRegsSoftmax + kPkRegsOut + kPkRegsRest <= 4 * kPkRegs, "the warpgroups' registers come out of the launch's");

template <int D>
struct PackedShape {
    static constexpr uint32_t kHalves = D / 64;                      // 64-element halves of a row
    static constexpr uint32_t kTile = kHalves * kPkTileBytes;        // a Q, K or V tile
    static constexpr uint32_t kStages = D == 64 ? 6 : 4;             // of K and V tiles, alternating
    static constexpr uint32_t kSmem = (2 + kStages) * kTile + 1024;  // and room to align
    // TMEM columns of row tile w: S, P and O.  At hd 64 P has columns of its own, and the next scores are
    // multiplied while the present ones become weights; at hd 128 there is room only over S.
    static constexpr bool kApart = D == 64;
    // One of so many pairs of exponentials is taken on the FMA pipe (0: none).  16384 keys, 16/2 heads, two
    // row tiles in step: hd 64 717 TFLOP/s without, 702 with one of 8, 685 with one of 4; hd 128, whose
    // products wait for the softmax, 1024 without, 1213 with one of 8, 1188 with one of 4.
    static constexpr int kPolyOf = D == 64 ? 0 : 8;
    static constexpr uint32_t s_col(uint32_t w) { return kApart ? w * 256 : w * 128; }
    static constexpr uint32_t p_col(uint32_t w) { return kApart ? w * 256 + 128 : w * 128; }
    static constexpr uint32_t o_col(uint32_t w) { return kApart ? w * 256 + 192 : 256 + w * 128; }
};

struct PackedArgs {
    void* out;
    const void* v;
    long long out_token, out_head, v_token, v_head;  // strides in elements
    const int32_t* offsets;
    uint32_t tokens, seqs, heads, kv_heads, hd;
    float scale_log2;
};

__device__ __forceinline__ uint32_t su32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok;
}

// Bounded wait; gives up early when another role has.
__device__ __forceinline__ bool mbar_wait_f(uint64_t* bar, uint32_t parity, volatile int* failed, uint32_t limit) {
    const uint32_t b = su32(bar);
    for (uint32_t it = 0; it < limit; ++it) {
        if (mbar_try(b, parity)) return true;
        if ((it & 31) == 31 && *failed) return false;
    }
    atomicMax(&g_packed_err, 1u);
    *failed = 1;
    return false;
}

// The drain of copies or products this thread issued, before the CTA may release what they touch.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < kPkSpin && !mbar_try(su32(bar), parity); ++it) {
    }
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar)) : "memory");
}

// One lane of the (converged) warp
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}

// Shared-memory matrix descriptors of tiles written by TMA with the 128-byte swizzle: rows of 128
// bytes, 8-row groups 1024 bytes apart.  K-major (Q, K): the next 16 elements of a row are 32 bytes on.
// MN-major (V): the next 16 keys are 2048 bytes on, the next 64 dims a tile half (16 KB).  addr16: the
// address in units of 16 bytes (below 2^14: shared memory).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr16) {
    return (uint64_t)(addr16 | (1u << 16)) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr16) {
    return (uint64_t)(addr16 | ((kPkTileBytes >> 4) << 16)) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// f32 accumulators, both operands f16 or both bf16; B K-major or MN-major.
template <bool BF16>
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_mn) {
    return (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((kPkRows >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(id), "r"(add));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(add));
}

// x = 64 * half elements: a multiple of 16 bytes
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, uint32_t half, uint32_t head, uint32_t token,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(half * 64), "r"(head), "r"(token), "r"(su32(bar))
        : "memory");
}

__device__ __forceinline__ void expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}

// 32 columns of this warp's 32 TMEM lanes: thread = lane.
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two f32 operations in one instruction.
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// 2^x for two x <= 9: x = n + f with n the nearest whole number (the low bits of x + 1.5 * 2^23),
// 2^f by the cubic with the least relative error on [-1/2, 1/2] (Remez exchange: 7.5e-5, below the
// weights' rounding to 16 bits), n added to its exponent.  Below 2^-127 that sum would be negative, and is cut
// to 0: what a row does not see (x = -inf) has no weight at all.  (bf16 has 2^-126 as a normal number, and
// times a V element of 1e38 it counts.)  x is cut at -250 first, so that n stays in the word.
__device__ __forceinline__ void ex2_poly(Pair xy, float& a, float& b) {
    float x, y;
    unpair(xy, x, y);
    xy = pair(fmaxf(x, -250.f), fmaxf(y, -250.f));
    const Pair big = pair(12582912.f, 12582912.f), nbig = pair(-12582912.f, -12582912.f), one = pair(-1.f, -1.f);
    const Pair n = add2(xy, big);
    const Pair f = fma2(add2(n, nbig), one, xy);
    Pair r = fma2(pair(0x1.c3f760p-5f, 0x1.c3f760p-5f), f, pair(0x1.f0de1ap-3f, 0x1.f0de1ap-3f));
    r = fma2(r, f, pair(0x1.62f31ap-1f, 0x1.62f31ap-1f));
    r = fma2(r, f, pair(0x1.fff692p-1f, 0x1.fff692p-1f));
    float nx, ny;
    unpair(n, nx, ny);
    unpair(r, a, b);
    a = __int_as_float(max(__float_as_int(a) + (__float_as_int(nx) << 23), 0));
    b = __int_as_float(max(__float_as_int(b) + (__float_as_int(ny) << 23), 0));
}

// Rows [begin, begin + len) of the packed tensors, the pair-th 256 of them, of one head; len 0: no more.
struct Item {
    uint32_t begin, len, pair, head;
};

// A 16-bit element whose exponent bits are all ones
template <bool BF16>
__device__ __forceinline__ bool not_finite16(uint32_t x) {
    constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
    return (x & e) == e;
}

}  // namespace

template <int D, bool BF16>
__global__ void __launch_bounds__(kPkThreads, 1)
    k_attn_packed(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, PackedArgs a) {
    using Sh = PackedShape<D>;
    constexpr uint32_t kStages = Sh::kStages, kTile = Sh::kTile, kHalves = Sh::kHalves;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t kv_full[kStages], kv_empty[kStages], v_raw[kPkClean], v_clean[kPkClean];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], s_full[2], p_full[2][2], o_full[2], l_full[2], o_empty[2], drain[2], lead;
    __shared__ __align__(8) uint64_t s_free[2], pv_done[2];  // S is in registers; P may be overwritten (kApart)
    __shared__ __align__(8) uint64_t it_full[kPkItems], it_empty[kPkItems];
    __shared__ Item s_item[kPkItems];
    __shared__ float s_inv[2][128];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int s_fail;
    // 1 + the last item of its parity in whose partly seen V tiles an element was not finite.  Two, as an output
    // warp may clean the next item's tiles while another has yet to look at this one's flag; before the flag's next
    // use, two items on, every thread has arrived on a barrier of the item between, behind its look.
    __shared__ uint32_t s_foul[kPkFoul];

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 32) {
        s_fail = 0;
        for (uint32_t i = 0; i < kPkFoul; ++i) s_foul[i] = 0;
        auto init = [](uint64_t* bar, uint32_t count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count));
        };
        for (uint32_t i = 0; i < kStages; ++i) {
            init(&kv_full[i], 1);
            init(&kv_empty[i], Sh::kApart ? 1 : 2);  // one thread's release, or both row tiles'
        }
        for (uint32_t i = 0; i < kPkClean; ++i) {
            init(&v_raw[i], 1);
            init(&v_clean[i], 128);
        }
        for (uint32_t i = 0; i < kPkItems; ++i) {
            init(&it_full[i], 1);
            init(&it_empty[i], 15);  // 8 softmax warps, 4 output warps, 2 of products, loads
        }
        init(&lead, 128);
        for (int i = 0; i < 2; ++i) {
            init(&q_full[i], 1);
            init(&q_empty[i], 1);
            init(&s_full[i], 1);
            init(&p_full[i][0], 128);
            init(&p_full[i][1], 128);
            init(&o_full[i], 1);
            init(&l_full[i], 128);
            init(&o_empty[i], 128);
            init(&drain[i], 1);
            init(&s_free[i], 128);
            init(&pv_done[i], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base, limit = g_packed_spin;
    const uint32_t smem = (su32(smem_raw) + 1023) & ~1023u;
    const uint32_t sq = smem, skv = smem + 2 * kTile;
    const uint32_t group = a.heads / a.kv_heads;
    auto wait = [&](uint64_t* bar, uint32_t phase) { return mbar_wait_f(bar, phase & 1, &s_fail, limit); };
    // The k-th item of this CTA, read by a whole warp or (one) by a single thread.
    auto next_item = [&](uint32_t k, Item& it, bool one) {
        bool ok = wait(&it_full[k % kPkItems], k / kPkItems);
        if (!one) ok = __all_sync(0xffffffffu, ok);
        if (!ok) return false;
        it = s_item[k % kPkItems];
        if (!one) __syncwarp();
        if (one || lane == 0) mbar_arrive(&it_empty[k % kPkItems]);
        return it.len != 0;
    };
    // key tiles of each row tile: up to the one on its diagonal
    auto tiles0 = [](const Item& it) { return 2 * it.pair + 1; };
    auto tiles1 = [](const Item& it) { return it.pair * 256 + 128 < it.len ? 2 * it.pair + 2 : 0; };

    if (warp >= 4 && warp < 12) {
        // ---- softmax of row tile w: thread = row ---------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPkRegsSoftmax));
        const uint32_t w = (warp >> 2) - 1, row = tid & 127;
        const uint32_t lanes = (32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + Sh::s_col(w), tp = tmem + lanes + Sh::p_col(w), to = tmem + lanes + Sh::o_col(w);
        const float c = a.scale_log2;
        uint32_t steps = 0, done = 0;  // key tiles and items of this row tile so far
        bool ok = true;
        Item it;
        for (uint32_t k = 0; ok && next_item(k, it, false); ++k) {
            const uint32_t tiles = w ? tiles1(it) : tiles0(it);
            if (!tiles) continue;
            float m = 0.f, mc = 0.f;  // the reference, and what it takes off a score in the exponent
            Pair l2 = pair(0.f, 0.f), l3 = l2;
            // 64 scores from column `at` on, key columns beyond the row's own unseen where that is the diagonal
            auto mask = [&](uint32_t (&s)[2][32], uint32_t at) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (at + i > row) s[i / 32][i % 32] = 0xff800000u;
            };
            auto largest = [&](const uint32_t (&s)[2][32]) {
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t* q = &s[i / 2][i % 2 * 16];
                    top[i] = __uint_as_float(q[0]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2) top[i] = max3(top[i], __uint_as_float(q[e]), __uint_as_float(q[e + 1]));
                    top[i] = max3(top[i], __uint_as_float(q[15]), top[i]);
                }
                return max3(max3(top[0], top[1], top[2]), top[3], top[0]);
            };
            // The reference after key tile `tile`'s largest score mx.  NaN among the scores stays NaN in the maximum,
            // and infinity makes one, as inf - inf: the whole row is NaN then, whichever way its exponentials are
            // taken.  Where the reference moves, the row's sums so far are scaled, those in TMEM once the product
            // of `before` steps is complete (hd 128: it is, as the scores were issued behind it).
            auto settle = [&](float mx, uint32_t tile, uint32_t before) {
                if (mx == INFINITY) mx = __int_as_float(0x7fffffff);
                const bool move = tile == 0 || !((mx - m) * c <= 8.f);
                if (tile == 0) {
                    m = mx;
                } else if (__any_sync(0xffffffffu, move)) {  // each row by itself: none depends on its neighbours
                    const float m_new = move ? max3(m, mx, mx) : m, f = move && m_new != -INFINITY ? ex2((m - m_new) * c) : 1.f;
                    m = m_new;
                    float x, y;
                    unpair(l2, x, y);
                    l2 = pair(x * f, y * f);
                    unpair(l3, x, y);
                    l3 = pair(x * f, y * f);
                    if (Sh::kApart) {
                        if (!__all_sync(0xffffffffu, wait(&pv_done[w], before))) return false;
                        fence_after();
                    }
#pragma unroll 1
                    for (uint32_t d = 0; d < D; d += 16) {
                        uint32_t o[16];
                        tmem_ld16(o, to + d);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(to + d, o);
                    }
                }
                mc = m == -INFINITY ? 0.f : -m * c;
                return true;
            };
            // n weights in pairs, from pair i0 of 64 scores on, into p
            auto weights = [&](const uint32_t (&s)[2][32], int i0, uint32_t* p, int n) {
                const Pair cc = pair(c, c), mm = pair(mc, mc);
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const uint32_t e = 2 * (i0 + i);
                    const Pair t = fma2(pair(__uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1])), cc, mm);
                    float x, y;
                    if (Sh::kPolyOf && i % (Sh::kPolyOf ? Sh::kPolyOf : 1) == 1) {
                        ex2_poly(t, x, y);
                    } else {
                        unpair(t, x, y);
                        x = ex2(x);
                        y = ex2(y);
                    }
                    if (i & 1)
                        l3 = add2(l3, pair(x, y));
                    else
                        l2 = add2(l2, pair(x, y));
                    p[i] = pack2<BF16>(x, y);
                }
            };
            auto load = [&](uint32_t (&s)[2][32], uint32_t at) {
                tmem_ld32(s[0], ts + at);
                tmem_ld32(s[1], ts + at + 32);
            };
            uint32_t a0[2][32], a1[2][32], p[32];  // the two halves of a row's scores, and 64 weights
            for (uint32_t j = 0; j < tiles; ++j, ++steps) {
                ok = __all_sync(0xffffffffu, wait(&s_full[w], steps));
                if (!ok) break;
                fence_after();
                load(a0, 0);
                load(a1, 64);
                tmem_wait_ld();
                if (Sh::kApart) {
                    fence_before();
                    mbar_arrive(&s_free[w]);
                }
                if (j + 1 == tiles) {
                    mask(a0, 0);
                    mask(a1, 64);
                }
                const float mx = largest(a0);
                ok = settle(max3(mx, largest(a1), mx), j, steps - 1);
                if (!ok) break;
                weights(a0, 0, p, 32);
                if (Sh::kApart && steps) {  // the last weights have been used
                    ok = __all_sync(0xffffffffu, wait(&pv_done[w], steps - 1));
                    if (!ok) break;
                    fence_after();
                }
                tmem_st32(tp, p);
                weights(a1, 0, p, 16);
                if (!Sh::kApart) {  // the products of the first 64 keys begin under the last weights
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(&p_full[w][0]);
                }
                weights(a1, 16, p + 16, 16);
                tmem_st32(tp + 32, p);
                tmem_wait_st();
                fence_before();
                mbar_arrive(&p_full[w][1]);
                if (!Sh::kApart && w == 0 && j == 0 && tiles1(it)) mbar_arrive(&lead);
            }
            if (!ok) break;
            if (done) ok = __all_sync(0xffffffffu, wait(&o_empty[w], done - 1));  // the last item's sums have been read
            float x0, y0, x1, y1;
            unpair(l2, x0, y0);
            unpair(l3, x1, y1);
            s_inv[w][row] = 1.f / ((x0 + y0) + (x1 + y1));
            mbar_arrive(&l_full[w]);
            ++done;
        }
        tmem_wait_st();  // none in flight when TMEM is released, wherever the loop was left
    } else if (warp >= 12) {
        // ---- output, and the V tiles that some row sees only in part ------------------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPkRegsOut));
        const uint32_t row = tid & 127, lanes = (32 * (warp & 3)) << 16;
        uint32_t done[2] = {0, 0}, ring = 0, clean = 0;
        bool ok = true;
        Item it;
        for (uint32_t k = 0; ok && next_item(k, it, false); ++k) {
            const uint32_t n0 = tiles0(it), n1 = tiles1(it), n = max(n0, n1);
            for (uint32_t j = n0 - 1; j < n && ok; ++j, ++clean) {
                ok = wait(&v_raw[clean % kPkClean], clean / kPkClean);
                const uint32_t v = skv + ((ring + 2 * j + 1) % kStages) * kTile;
                for (uint32_t i = row; i < kTile / 16 && ok; i += 128) {
                    uint32_t x[4];
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                                 : "r"(v + i * 16)
                                 : "memory");
                    bool here = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (not_finite16<BF16>(x[e])) {
                            x[e] &= 0xFFFF0000u;
                            here = true;
                        }
                        if (not_finite16<BF16>(x[e] >> 16)) {
                            x[e] &= 0xFFFFu;
                            here = true;
                        }
                    }
                    if (here) {
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(v + i * 16), "r"(x[0]), "r"(x[1]), "r"(x[2]),
                                     "r"(x[3])
                                     : "memory");
                        s_foul[k % kPkFoul] = k + 1;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&v_clean[clean % kPkClean]);
                ok = ok && wait(&v_clean[clean % kPkClean], clean / kPkClean);  // every thread's part: the flag is settled
            }
            ok = __all_sync(0xffffffffu, ok);
            const bool foul = ok && *(volatile uint32_t*)&s_foul[k % kPkFoul] == k + 1;
            ring += 2 * n;
#pragma unroll
            for (uint32_t w = 0; w < 2; ++w) {
                if (!ok || (w && !n1)) break;
                ok = wait(&l_full[w], done[w]) && wait(&o_full[w], done[w]);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++done[w];
                fence_after();
                const float inv = s_inv[w][row];
                const uint32_t at = it.pair * 256 + w * 128 + row, to = tmem + lanes + Sh::o_col(w);
                const bool live = at < it.len;
                uint16_t* dst = static_cast<uint16_t*>(a.out) + (long long)(it.begin + at) * a.out_token + (long long)it.head * a.out_head;
#pragma unroll 1
                for (uint32_t d = 0; d < D; d += 64) {
                    // O is free for the next item as soon as it is in registers
                    uint32_t o[2][32];
                    tmem_ld32(o[0], to + d);
                    tmem_ld32(o[1], to + d + 32);
                    tmem_wait_ld();
                    if (d + 64 == D) {
                        fence_before();
                        mbar_arrive(&o_empty[w]);
                    }
                    if (foul && live) {
                        // elements that are not finite, of the keys of the last two tiles that this row sees
                        const uint16_t* v = static_cast<const uint16_t*>(a.v) + (long long)(it.head / group) * a.v_head;
                        for (uint32_t key = it.pair * 256; key <= at; ++key) {
                            const uint16_t* vr = v + (long long)(it.begin + key) * a.v_token + d;
#pragma unroll
                            for (int i = 0; i < 64; ++i)
                                if (d + i < a.hd && not_finite16<BF16>(vr[i]))
                                    o[i / 32][i % 32] = __float_as_uint(__uint_as_float(o[i / 32][i % 32]) +
                                                                        (BF16 ? __uint_as_float((uint32_t)vr[i] << 16)
                                                                              : __half2float(__ushort_as_half(vr[i]))));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 64; i += 8)
                        if (live && d + i < a.hd) {
                            const uint32_t* q = &o[i / 32][i % 32];
                            uint4 r;
                            r.x = pack2<BF16>(__uint_as_float(q[0]) * inv, __uint_as_float(q[1]) * inv);
                            r.y = pack2<BF16>(__uint_as_float(q[2]) * inv, __uint_as_float(q[3]) * inv);
                            r.z = pack2<BF16>(__uint_as_float(q[4]) * inv, __uint_as_float(q[5]) * inv);
                            r.w = pack2<BF16>(__uint_as_float(q[6]) * inv, __uint_as_float(q[7]) * inv);
                            *reinterpret_cast<uint4*>(dst + d + i) = r;
                        }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPkRegsRest));
        // The product warps run their loops as a whole, on values that the compiler sees to be the same in all
        // lanes (votes, shuffles from lane 0), so that descriptors stay in uniform registers; one elected
        // lane issues.  A tcgen05 operand that comes from one lane's own register costs some 15 clocks.
        const bool lead_lane = elect_one();
        auto wait_all = [&](uint64_t* bar, uint32_t phase) { return (bool)__all_sync(0xffffffffu, wait(bar, phase)); };
        auto next_all = [&](uint32_t k, uint32_t* n0, uint32_t* n1) {  // the key tiles of the k-th item's row tiles
            Item it{};
            const bool got = next_item(k, it, false);
            *n0 = __shfl_sync(0xffffffffu, got ? tiles0(it) : 0u, 0);
            *n1 = __shfl_sync(0xffffffffu, got ? tiles1(it) : 0u, 0);
            return *n0 != 0;
        };
        if (Sh::kApart && warp == 0) {
            // ---- scores of both row tiles, ahead of the softmax by a key tile ------------------------------------
            uint32_t scores[2] = {0, 0}, done[2] = {0, 0}, stage = 0, round = 0;  // of the ring's next K tile
            bool ok = true;
            uint32_t n0, n1;
            for (uint32_t k = 0; ok && next_all(k, &n0, &n1); ++k) {
                const uint32_t n = max(n0, n1);
                for (uint32_t j = 0; j < n && ok; ++j) {
                    const uint32_t klo = (skv + stage * kTile) >> 4;
                    ok = wait_all(&kv_full[stage], round);
#pragma unroll
                    for (uint32_t w = 0; w < 2; ++w) {
                        const uint32_t mine = w ? n1 : n0, qlo = (sq + w * kTile) >> 4;
                        if (!ok || j >= mine) continue;
                        if (j == 0) ok = wait_all(&q_full[w], done[w]);
                        if (ok && scores[w]) ok = wait_all(&s_free[w], scores[w] - 1);
                        if (!ok) break;
                        ++scores[w];
                        fence_after();
                        if (lead_lane) {
#pragma unroll
                            for (uint32_t i = 0; i < D / 16; ++i)
                                mma_ss(tmem + Sh::s_col(w), desc_k(qlo + 2 * i), desc_k(klo + 2 * i), idesc<BF16>(128, false), i);
                            commit(&s_full[w]);
                            if (j + 1 == mine) commit(&q_empty[w]);
                        }
                        done[w] += j + 1 == mine;
                    }
                    if (lead_lane) commit(&kv_empty[stage]);
                    stage += 2;
                    if (stage == kStages) {
                        stage = 0;
                        ++round;
                    }
                }
            }
            if (lead_lane) {
                commit(&drain[0]);
                mbar_drain(&drain[0], 0);
            }
        } else if (Sh::kApart && warp == 3) {
            // ---- weights times V, of both row tiles ------------------------------------------------------------------
            uint32_t steps[2] = {0, 0}, done[2] = {0, 0}, clean = 0, stage = 1, round = 0;  // of the ring's next V tile
            bool ok = true;
            uint32_t n0, n1;
            for (uint32_t k = 0; ok && next_all(k, &n0, &n1); ++k) {
                const uint32_t n = max(n0, n1);
                for (uint32_t j = 0; j < n && ok; ++j) {
                    const uint32_t vlo = (skv + stage * kTile) >> 4;
                    if (j >= n0 - 1) {
                        ok = wait_all(&v_clean[clean % kPkClean], clean / kPkClean);
                        ++clean;
                    } else {
                        ok = wait_all(&kv_full[stage], round);
                    }
#pragma unroll
                    for (uint32_t w = 0; w < 2; ++w) {
                        const uint32_t mine = w ? n1 : n0;
                        if (!ok || j >= mine) continue;
                        if (j == 0 && done[w]) ok = wait_all(&o_empty[w], done[w] - 1);
                        ok = ok && wait_all(&p_full[w][1], steps[w]);
                        if (!ok) break;
                        ++steps[w];
                        fence_after();
                        if (lead_lane) {
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i)
                                mma_ts(tmem + Sh::o_col(w), tmem + Sh::p_col(w) + 8 * i, desc_mn(vlo + i * 128), idesc<BF16>(D, true), j | i);
                            commit(&pv_done[w]);
                            if (j + 1 == mine) commit(&o_full[w]);
                        }
                        done[w] += j + 1 == mine;
                    }
                    if (lead_lane) commit(&kv_empty[stage]);
                    stage += 2;
                    if (stage > kStages) {
                        stage = 1;
                        ++round;
                    }
                }
            }
            // every product complete before TMEM and the tiles are released
            if (lead_lane) {
                commit(&drain[1]);
                mbar_drain(&drain[1], 0);
            }
        } else if (warp == 0 || warp == 3) {
            // ---- the products of row tile w ------------------------------------------------------------------------------
            const uint32_t w = __shfl_sync(0xffffffffu, warp == 3 ? 1u : 0u, 0);
            uint32_t steps = 0, done = 0, clean = 0;
            uint32_t stage = 0, round = 0;  // of the ring's next tile
            const uint32_t qlo = (sq + w * kTile) >> 4;
            const uint32_t ts = tmem + Sh::s_col(w), tp = tmem + Sh::p_col(w), to = tmem + Sh::o_col(w);
            auto advance = [&]() {
                if (++stage == kStages) {
                    stage = 0;
                    ++round;
                }
            };
            auto full = [&]() { return wait_all(&kv_full[stage], round); };
            // S = Q K^T with the ring's next tile, which is there and then released
            auto qk = [&](bool last) {
                const uint32_t klo = (skv + stage * kTile) >> 4;
                if (lead_lane) {
#pragma unroll
                    for (uint32_t i = 0; i < D / 16; ++i) {
                        const uint32_t off = ((i / 4) * kPkTileBytes + (i % 4) * 32) >> 4;
                        mma_ss(ts, desc_k(qlo + off), desc_k(klo + off), idesc<BF16>(128, false), i);
                    }
                    commit(&s_full[w]);
                    commit(&kv_empty[stage]);
                    if (last) commit(&q_empty[w]);
                }
                advance();
            };
            bool ok = true;
            uint32_t n0, n1;
            for (uint32_t k = 0; ok && next_all(k, &n0, &n1); ++k) {
                const uint32_t n = max(n0, n1), mine = w ? n1 : n0;
                if (mine) {
                    ok = wait_all(&q_full[w], done) && full();
                    // Row tile 1 sets out when tile 0's first weights are done: in step, the two would
                    // want the same pipes at the same time and leave them idle together.
                    if (ok && w) ok = wait_all(&lead, done);
                    if (!ok) break;
                    fence_after();
                    qk(mine == 1);
                }
                for (uint32_t j = 0; j < mine; ++j, ++steps) {
                    // V tile j, then K tile j + 1 of the ring; what is there early is waited for early
                    const uint32_t vlo = (skv + stage * kTile) >> 4, v_stage = stage;
                    const bool more = j + 1 < mine;
                    ok = j >= n0 - 1 ? wait_all(&v_clean[(clean + j - (n0 - 1)) % kPkClean], (clean + j - (n0 - 1)) / kPkClean) : full();
                    advance();
                    ok = ok && (!more || full());
                    if (ok && j == 0 && done) ok = wait_all(&o_empty[w], done - 1);
                    ok = ok && wait_all(&p_full[w][0], steps);
                    if (!ok) break;
                    fence_after();
                    if (lead_lane) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) mma_ts(to, tp + 8 * i, desc_mn(vlo + i * 128), idesc<BF16>(D, true), j | i);
                    }
                    ok = wait_all(&p_full[w][1], steps);
                    if (!ok) break;
                    fence_after();
                    if (lead_lane) {
#pragma unroll
                        for (uint32_t i = 4; i < 8; ++i) mma_ts(to, tp + 8 * i, desc_mn(vlo + i * 128), idesc<BF16>(D, true), 1);
                    }
                    if (more)
                        qk(j + 2 == mine);
                    else if (lead_lane)
                        commit(&o_full[w]);
                    if (lead_lane) commit(&kv_empty[v_stage]);
                }
                if (!ok) break;
                done += mine != 0;
                // tiles that only the other row tile uses: released once they are there, in the ring's order
                for (uint32_t j = 2 * mine; j < 2 * n && ok; ++j) {
                    ok = full();
                    if (ok && lead_lane) mbar_arrive(&kv_empty[stage]);
                    advance();
                }
                clean += n - (n0 - 1);
            }
            // every product complete before TMEM and the tiles are released
            if (lead_lane) {
                commit(&drain[w]);
                mbar_drain(&drain[w], 0);
            }
        } else if (warp == 1) {
            // ---- loads: one thread -----------------------------------------------------------------------------
            if (lane == 0) {
                uint32_t ring = 0, clean = 0, sent_q[2] = {0, 0};
                auto load_q = [&](const Item& it, uint32_t w) {
                    if (sent_q[w] && !wait(&q_empty[w], sent_q[w] - 1)) return false;
                    ++sent_q[w];
                    expect_tx(&q_full[w], kTile);
#pragma unroll
                    for (uint32_t h = 0; h < kHalves; ++h)
                        tma_tile(sq + w * kTile + h * kPkTileBytes, &qmap, h, it.head, it.begin + it.pair * 256 + w * 128, &q_full[w]);
                    return true;
                };
                // tile t of the ring: of K, or of V with a barrier of its own where some row sees it in part
                auto load_kv = [&](const Item& it, uint32_t t, uint32_t j, const CUtensorMap* map, uint64_t* bar) {
                    if (t >= kStages && !wait(&kv_empty[t % kStages], t / kStages - 1)) return false;
                    expect_tx(bar, kTile);
#pragma unroll
                    for (uint32_t h = 0; h < kHalves; ++h)
                        tma_tile(skv + (t % kStages) * kTile + h * kPkTileBytes, map, h, it.head / group, it.begin + j * 128, bar);
                    return true;
                };
                bool ok = true;
                Item it;
                for (uint32_t k = 0; ok && next_item(k, it, true); ++k) {
                    const uint32_t n0 = tiles0(it), n1 = tiles1(it), n = max(n0, n1);
                    ok = load_q(it, 0);
                    for (uint32_t j = 0; j < n && ok; ++j) {
                        ok = load_kv(it, ring, j, &kmap, &kv_full[ring % kStages]);
                        if (!ok) break;
                        ++ring;
                        // Q of row tile 1 behind K tile 0: the products wait for that one first
                        if (j == 0 && n1) ok = load_q(it, 1);
                        if (!ok) break;
                        // (a V tile on a barrier of its own keeps its stage's in step with an empty phase)
                        if (j >= n0 - 1) {
                            ok = load_kv(it, ring, j, &vmap, &v_raw[clean % kPkClean]);
                            if (ok) mbar_arrive(&kv_full[ring % kStages]);
                            clean += ok;
                        } else {
                            ok = load_kv(it, ring, j, &vmap, &kv_full[ring % kStages]);
                        }
                        ring += ok;
                    }
                }
                // no copy may still be landing when the CTA releases its shared memory: the last of each barrier
                for (uint32_t w = 0; w < 2; ++w)
                    if (sent_q[w]) mbar_drain(&q_full[w], (sent_q[w] - 1) & 1);
                for (uint32_t i = ring > kStages ? ring - kStages : 0; i < ring; ++i) mbar_drain(&kv_full[i % kStages], (i / kStages) & 1);
                for (uint32_t i = clean > kPkClean ? clean - kPkClean : 0; i < clean; ++i) mbar_drain(&v_raw[i % kPkClean], (i / kPkClean) & 1);
            }
        } else {
            // ---- items: pairs of row tiles in descending order, heads innermost -----------------------------------
            auto tiles_of = [&](uint32_t s, uint32_t* begin, uint32_t* len) -> uint32_t {  // of prompt s, in pairs
                if (s >= a.seqs) return 0;
                const uint32_t b = (uint32_t)min(max(a.offsets[s], 0), (int32_t)a.tokens);
                const uint32_t e = (uint32_t)min(max(a.offsets[s + 1], 0), (int32_t)a.tokens);
                *begin = b;
                *len = e > b ? e - b : 0;
                return (*len + 255) / 256;
            };
            uint32_t my_begin = 0, my_len = 0, most = 0, x, y;
            const uint32_t my_tiles = tiles_of(lane, &my_begin, &my_len);  // the first 32 prompts stay at hand
            for (uint32_t s = lane; s < a.seqs; s += 32) most = max(most, s < 32 ? my_tiles : tiles_of(s, &x, &y));
            most = __reduce_max_sync(0xffffffffu, most);
            // items of one head whose pair number is p or more
            auto at_least = [&](uint32_t p) {
                uint32_t sum = my_tiles > p ? my_tiles - p : 0;
                for (uint32_t s = lane + 32; s < a.seqs; s += 32) {
                    const uint32_t t = tiles_of(s, &x, &y);
                    sum += t > p ? t - p : 0;
                }
                return __reduce_add_sync(0xffffffffu, sum);
            };
            const unsigned long long total = (unsigned long long)at_least(0) * a.heads;
            for (uint32_t k = 0;; ++k) {
                const uint32_t c = k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
                const unsigned long long i = (unsigned long long)k * gridDim.x + c;
                Item it{0, 0, 0, 0};
                if (i < total) {
                    const uint32_t t = (uint32_t)(i / a.heads);
                    it.head = (uint32_t)(i % a.heads);
                    uint32_t lo = 0, hi = most;  // at_least(lo) > t >= at_least(hi)
                    uint32_t above = 0;          // at_least(hi)
                    while (hi - lo > 1) {
                        const uint32_t mid = (lo + hi) / 2, n = at_least(mid);
                        if (n > t) {
                            lo = mid;
                        } else {
                            hi = mid;
                            above = n;
                        }
                    }
                    it.pair = lo;
                    uint32_t r = t - above;  // the r-th prompt with more than `lo` pairs
                    for (uint32_t s0 = 0; s0 < a.seqs; s0 += 32) {
                        uint32_t b = my_begin, l = my_len, n = my_tiles;
                        if (s0) n = tiles_of(s0 + lane, &b, &l);
                        const uint32_t has = __ballot_sync(0xffffffffu, n > lo), count = __popc(has);
                        if (r < count) {
                            const uint32_t src = __fns(has, 0, r + 1);
                            it.begin = __shfl_sync(0xffffffffu, b, src);
                            it.len = __shfl_sync(0xffffffffu, l, src);
                            break;
                        }
                        r -= count;
                    }
                }
                bool ok = true;
                if (k >= kPkItems) ok = __all_sync(0xffffffffu, wait(&it_empty[k % kPkItems], k / kPkItems - 1));
                if (!ok) break;
                if (lane == 0) {
                    s_item[k % kPkItems] = it;
                    mbar_arrive(&it_full[k % kPkItems]);
                }
                __syncwarp();
                if (i >= total) break;
            }
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ---- launches -----------------------------------------------------------------------------------

// cuTensorMapEncodeTiled, looked up through the runtime so the library needs no link-time driver
// dependency.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// [tokens][heads][hd] 16-bit elements in boxes of 128 tokens x one head x 64 elements; what lies outside
// (tokens behind the last, elements behind hd) reads as 0.
static bool tile_map(CUtensorMap* map, bool bf16, const void* p, uint32_t hd, uint32_t heads, uint32_t tokens, long long token,
                     long long head) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[3] = {hd, heads, tokens};
    // (an axis of one entry has no step; any valid stride will do)
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head : hd) * 2, (cuuint64_t)(tokens > 1 ? token : hd) * 2};
    const cuuint32_t box[3] = {64, 1, 128}, unit[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims,
              strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
static enx_status launch_packed(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PackedArgs& a,
                                cudaStream_t st) {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];  // per device: the kernel's attributes are set and its registers suffice
    int dev = 0;
    ENX_CUDA(cudaGetDevice(&dev));
    if (dev >= kDevices || !known[dev].load(std::memory_order_acquire)) {
        cudaFuncAttributes f{};
        ENX_CUDA(cudaFuncGetAttributes(&f, k_attn_packed<D, BF16>));
        // the warpgroups' shares are drawn from what the block was launched with: less would wait for ever
        if (f.numRegs < kPkRegs) return fail(ENX_ERR_STATE, "enx_attn_packed: built with too few registers");
        ENX_CUDA(cudaFuncSetAttribute(k_attn_packed<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)PackedShape<D>::kSmem));
        if (dev < kDevices) known[dev].store(1, std::memory_order_release);
    }
    // a CTA per SM, or as many as there can be items
    const uint64_t most = ((uint64_t)a.tokens / 256 + a.seqs) * a.heads;
    const uint32_t grid = (uint32_t)(most < 148 ? most : 148);
    k_attn_packed<D, BF16><<<grid, kPkThreads, PackedShape<D>::kSmem, st>>>(q, k, v, a);
    ENX_CUDA(cudaGetLastError());
    return ENX_OK;
}

cudaError_t packed_set_spin(uint32_t spins) {
    const uint32_t v = spins ? spins : kPkSpin;
    return cudaMemcpyToSymbol(g_packed_spin, &v, sizeof(v));
}

cudaError_t packed_take_error(uint32_t* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_packed_err, sizeof(*code));
    const uint32_t zero = 0;
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_packed_err, &zero, sizeof(zero));
    return e;
}

}  // namespace enx

using namespace enx;

extern "C" enx_status enx_attn_packed(const void* q, const void* k, const void* v, void* out, const int64_t* strides,
                                      const int32_t* offsets, uint32_t seqs, uint32_t tokens, uint32_t heads, uint32_t kv_heads,
                                      uint32_t head_dim, uint32_t dtype, float scale, void* stream) {
    if (dtype != ENX_F16 && dtype != ENX_BF16) return fail(ENX_ERR_INVALID, "enx_attn_packed: dtype must be ENX_F16 or ENX_BF16");
    if (head_dim == 0 || head_dim % 8 || head_dim > 128)
        return fail(ENX_ERR_INVALID, "enx_attn_packed: head_dim must be a multiple of 8, at most 128");
    if (kv_heads == 0 || heads == 0 || heads % kv_heads)
        return fail(ENX_ERR_INVALID, "enx_attn_packed: heads must be a multiple of kv_heads");
    if (heads > 65535) return fail(ENX_ERR_RANGE, "enx_attn_packed: at most 65535 heads");
    // (a prompt of 2^24 tokens keeps the roles of a CTA waiting for one another within the waits' limit)
    if (tokens > (1u << 24) || seqs > (1u << 16)) return fail(ENX_ERR_RANGE, "enx_attn_packed: at most 2^24 tokens and 65536 prompts");
    if (!(scale > 0.f)) return fail(ENX_ERR_INVALID, "enx_attn_packed: scale must be positive");
    if (seqs == 0 || tokens == 0) return ENX_OK;
    if (!q || !k || !v || !out || !strides || !offsets) return fail(ENX_ERR_INVALID, "enx_attn_packed: null pointer");
    uintptr_t any = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                    reinterpret_cast<uintptr_t>(out);
    for (int i = 0; i < 8; ++i) {
        const bool used = i % 2 ? (i == 1 || i == 7 ? heads : kv_heads) > 1 : tokens > 1;
        if (used && (strides[i] <= 0 || strides[i] >= (1ll << 38)))
            return fail(ENX_ERR_RANGE, "enx_attn_packed: strides must be positive and below 2^38");
        if (used) any |= (uintptr_t)strides[i] * 2;
    }
    if (any % 16)
        return fail(ENX_ERR_INVALID, "enx_attn_packed: rows must start on 16 bytes (pointers, token and head strides)");
    const bool bf16 = dtype == ENX_BF16;
    CUtensorMap qm, km, vm;
    if (!tile_map(&qm, bf16, q, head_dim, heads, tokens, strides[0], strides[1]) ||
        !tile_map(&km, bf16, k, head_dim, kv_heads, tokens, strides[2], strides[3]) ||
        !tile_map(&vm, bf16, v, head_dim, kv_heads, tokens, strides[4], strides[5]))
        return fail(ENX_ERR_CUDA, "enx_attn_packed: cuTensorMapEncodeTiled refused a tensor");
    PackedArgs a{out, v, strides[6], strides[7], strides[4], strides[5], offsets, tokens, seqs, heads, kv_heads, head_dim,
                 scale * 1.4426950408889634f};
    if (head_dim <= 64)
        return bf16 ? launch_packed<64, true>(qm, km, vm, a, as_stream(stream))
                    : launch_packed<64, false>(qm, km, vm, a, as_stream(stream));
    return bf16 ? launch_packed<128, true>(qm, km, vm, a, as_stream(stream))
                : launch_packed<128, false>(qm, km, vm, a, as_stream(stream));
}
