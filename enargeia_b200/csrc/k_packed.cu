// Causal attention over whole prompts packed one behind another, with grouped heads, in f16 or bf16, on
// the 5th-generation tensor cores (tcgen05, TMEM accumulators).
//
// out[i] = sum_j softmax_j(scale * q[i].k[j]) v[j] over the keys j <= i of token i's own prompt.
//
// A CTA owns 256 consecutive queries of one prompt and head, as two tiles of 128 rows that take turns:
// while one warpgroup turns the first tile's scores into weights, the tensor cores multiply for the
// second.  Keys go by in tiles of 128, counted from the prompt's start like the rows, so that of each
// row tile only the last key tile needs a mask.  Per key tile and row tile:
//
//   S (TMEM, f32) = Q K^T           kind::f16, M = N = 128, both operands K-major from shared memory
//   p = 2^(scale' (s - m)), to TMEM over S, in 16 bits
//   O (TMEM, f32) += P V            A from TMEM, V MN-major from shared memory as it lies in memory
//
// m, a row's reference, starts as the first key tile's maximum and moves only when a score passes it by
// more than 2^8 in its weight; then the warpgroup rescales its rows of O in TMEM, which is rare.  Sums
// are f32.  Weights are rounded to the inputs' 16 bits for the product, as the output is.
//
// Bound: one exponential per score against 4 hd multiply-adds.  16 a clock and SM make 1024 clocks per
// 128 x 128 scores, the products 512 at hd 64 and 1024 at hd 128.
//
// Warp roles, synchronised by mbarriers with bounded waits:
//   warps 0-3, 4-7  softmax of row tile 0 and 1 (thread = row), then its output
//   warp 8          TMEM; lane 0 issues all products
//   warp 9          lane 0 loads Q, K and V tiles by TMA (128-byte swizzle; 64-element halves of a row)
//   warps 10, 11    look through the V tiles that some row sees only in part (see below)
//
// A weight of zero times a V element that is not finite would be NaN.  The last two key tiles of a CTA
// are the only ones that hold keys which some row does not see, so in those the helper warps replace such
// elements by zeros before the product, and where there were any, each row adds those that it does see
// when it writes its output.

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
constexpr uint32_t kPkThreads = 384;
constexpr uint32_t kPkTileBytes = 128 * 128;  // 128 rows of 64 16-bit elements
constexpr int kPkRegs = 168, kPkRegsSoftmax = 224, kPkRegsRest = 56;
static_assert(2 * kPkRegsSoftmax + kPkRegsRest <= 3 * kPkRegs, "the warpgroups' registers come out of the launch's");

template <int D>
struct PackedShape {
    static constexpr uint32_t kHalves = D / 64;                      // 64-element halves of a row
    static constexpr uint32_t kTile = kHalves * kPkTileBytes;        // a Q, K or V tile
    static constexpr uint32_t kStages = D == 64 ? 6 : 4;             // of K and V tiles, alternating
    static constexpr uint32_t kSmem = (2 + kStages) * kTile + 1024;  // and room to align
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

// Shared-memory matrix descriptors of tiles written by TMA with the 128-byte swizzle: rows of 128
// bytes, 8-row groups 1024 bytes apart.  K-major (Q, K): the next 16 elements of a row are 32 bytes on.
// MN-major (V): the next 16 keys are 2048 bytes on, the next 64 dims a tile half (16 KB).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kPkTileBytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
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
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
    constexpr uint32_t kTmemO = 256;  // columns: S (and P) of the two row tiles, then O of each
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full, kv_full[kStages], kv_empty[kStages], v_raw[2], v_clean[2], s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tmem_base, s_seq[3];
    __shared__ volatile int s_fail;
    __shared__ int s_foul;  // a V element that is not finite among the last two key tiles

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head = blockIdx.y;

    // ---- which prompt and which 256 rows: tile blockIdx.x of all prompts' tiles, long ones first ------
    if (warp == 0) {
        uint32_t before = 0, found = 0, begin = 0, len = 0, back = 0;
        for (uint32_t s0 = 0; s0 < a.seqs && !found; s0 += 32) {
            const uint32_t s = s0 + lane;
            uint32_t b = 0, n = 0;
            if (s < a.seqs) {
                b = (uint32_t)min(max(a.offsets[s], 0), (int32_t)a.tokens);
                const uint32_t e = (uint32_t)min(max(a.offsets[s + 1], 0), (int32_t)a.tokens);
                n = e > b ? e - b : 0;
            }
            const uint32_t tiles = (n + 255) / 256;
            uint32_t incl = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= (uint32_t)o) incl += up;
            }
            const uint32_t lo = before + incl - tiles;
            const uint32_t hit = __ballot_sync(0xffffffffu, blockIdx.x >= lo && blockIdx.x < lo + tiles);
            if (hit) {
                const int src = __ffs(hit) - 1;
                begin = __shfl_sync(0xffffffffu, b, src);
                len = __shfl_sync(0xffffffffu, n, src);
                back = blockIdx.x - __shfl_sync(0xffffffffu, lo, src);
                found = 1;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            s_seq[0] = begin;
            s_seq[1] = found ? len : 0;
            s_seq[2] = found ? (len + 255) / 256 - 1 - back : 0;
        }
    }
    if (tid == 32) {
        s_fail = 0;
        s_foul = 0;
        auto init = [](uint64_t* bar, uint32_t count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count));
        };
        init(&q_full, 1);
        for (uint32_t i = 0; i < kStages; ++i) {
            init(&kv_full[i], 1);
            init(&kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            init(&v_raw[i], 1);
            init(&v_clean[i], 64);
            init(&s_full[i], 1);
            init(&p_full[i], 128);
            init(&o_full[i], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const uint32_t begin = s_seq[0], len = s_seq[1], pair_tile = s_seq[2];
    if (len == 0) return;  // the grid covers the most tiles that the offsets could make
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base, limit = g_packed_spin;
    const uint32_t smem = (su32(smem_raw) + 1023) & ~1023u;
    const uint32_t sq = smem, skv = smem + 2 * kTile;
    const uint32_t kvh = head / (a.heads / a.kv_heads);
    const uint32_t first_row = pair_tile * 256;  // of the prompt
    // key tiles of each row tile: up to the one on its diagonal
    const uint32_t n0 = 2 * pair_tile + 1, n1 = first_row + 128 < len ? n0 + 1 : 0, n = max(n0, n1);

    if (warp < 8) {
        // ---- softmax of row tile w: thread = row ---------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPkRegsSoftmax));
        const uint32_t w = warp >> 2, row = tid & 127, tiles = w ? n1 : n0;
        const uint32_t lanes = (32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + w * 128, to = tmem + lanes + kTmemO + w * D;
        const float c = a.scale_log2;
        float m = 0.f;
        Pair l2 = pair(0.f, 0.f), l3 = l2;
        bool ok = true;
        for (uint32_t j = 0; j < tiles; ++j) {
            if (!mbar_wait_f(&s_full[w], j & 1, &s_fail, limit)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld32(s[i], ts + 32 * i);
            tmem_wait_ld();
            if (j + 1 == tiles) {  // the diagonal: key column > row is not seen
#pragma unroll
                for (int i = 0; i < 128; ++i)
                    if ((uint32_t)i > row) s[i / 32][i % 32] = 0xff800000u;
            }
            float top[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                top[i] = __uint_as_float(s[i][0]);
#pragma unroll
                for (int k = 1; k < 32; ++k) top[i] = fmaxf(top[i], __uint_as_float(s[i][k]));
            }
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (j == 0) {
                m = mx;
            } else if (__any_sync(0xffffffffu, (mx - m) * c > 8.f)) {
                const float m_new = fmaxf(m, mx), f = m_new == -INFINITY ? 1.f : ex2((m - m_new) * c);
                m = m_new;
                float x, y;
                unpair(l2, x, y);
                l2 = pair(x * f, y * f);
                unpair(l3, x, y);
                l3 = pair(x * f, y * f);
                // the product of the last key tile is complete: this tile's scores were issued after it
#pragma unroll 1
                for (uint32_t k = 0; k < D; k += 32) {
                    uint32_t o[32];
                    tmem_ld32(o, to + k);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st32(to + k, o);
                }
            }
            const float mc = m == -INFINITY ? 0.f : -m * c;
            const Pair cc = pair(c, c), mm = pair(mc, mc);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const uint32_t e = 64 * h + 2 * i;
                    float x, y;
                    unpair(fma2(pair(__uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1])), cc, mm), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    if (i & 1)
                        l3 = add2(l3, pair(x, y));
                    else
                        l2 = add2(l2, pair(x, y));
                    p[i] = pack2<BF16>(x, y);
                }
                tmem_st32(ts + 32 * h, p);
            }
            tmem_wait_st();
            fence_before();
            mbar_arrive(&p_full[w]);
        }
        if (tiles && ok) {
            if (!mbar_wait_f(&o_full[w], 0, &s_fail, limit)) ok = false;
            for (uint32_t i = 0; i < tiles - (n0 - 1); ++i)  // long since complete: orders the read of s_foul
                if (!mbar_wait_f(&v_clean[i], 0, &s_fail, limit)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
        }
        if (tiles && ok) {
            fence_after();
            float x0, y0, x1, y1;
            unpair(l2, x0, y0);
            unpair(l3, x1, y1);
            const float inv = 1.f / ((x0 + y0) + (x1 + y1));
            const uint32_t at = first_row + w * 128 + row;
            const bool live = at < len;
            uint16_t* dst = static_cast<uint16_t*>(a.out) + (long long)(begin + at) * a.out_token + (long long)head * a.out_head;
#pragma unroll 1
            for (uint32_t k = 0; k < D; k += 32) {
                uint32_t o[32];
                tmem_ld32(o, to + k);
                tmem_wait_ld();
                if (s_foul && live) {
                    // elements that are not finite, of the keys of the last two tiles that this row sees
                    const uint16_t* v = static_cast<const uint16_t*>(a.v) + (long long)kvh * a.v_head;
                    for (uint32_t key = first_row; key <= at; ++key) {
                        const uint16_t* vr = v + (long long)(begin + key) * a.v_token + k;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (k + i < a.hd && not_finite16<BF16>(vr[i]))
                                o[i] = __float_as_uint(__uint_as_float(o[i]) +
                                                       (BF16 ? __uint_as_float((uint32_t)vr[i] << 16)
                                                             : __half2float(__ushort_as_half(vr[i]))));
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    if (live && k + i < a.hd) {
                        uint4 r;
                        r.x = pack2<BF16>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                        r.y = pack2<BF16>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                        r.z = pack2<BF16>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                        r.w = pack2<BF16>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                        *reinterpret_cast<uint4*>(dst + k + i) = r;
                    }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPkRegsRest));
        // Stage and phase of the i-th tile of the ring: K tile j is 2j, V tile j is 2j + 1.  The V tiles from
        // n0 - 1 on, whose stages are not used again, land on barriers of their own, for the helpers.
        auto full_wait = [&](uint32_t i) { return mbar_wait_f(&kv_full[i % kStages], (i / kStages) & 1, &s_fail, limit); };
        if (warp == 8) {
            // ---- all products: one thread ------------------------------------------------------------------
            if (lane == 0) {
                auto qk = [&](uint32_t w, uint32_t j) {
                    const uint32_t k = skv + ((2 * j) % kStages) * kTile, q = sq + w * kTile;
#pragma unroll
                    for (uint32_t i = 0; i < D / 16; ++i) {
                        const uint32_t off = (i / 4) * kPkTileBytes + (i % 4) * 32;
                        mma_ss(tmem + w * 128, desc_k(q + off), desc_k(k + off), idesc<BF16>(128, false), i);
                    }
                };
                auto pv = [&](uint32_t w, uint32_t j) {
                    const uint32_t v = skv + ((2 * j + 1) % kStages) * kTile;
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        mma_ts(tmem + kTmemO + w * D, tmem + w * 128 + 8 * i, desc_mn(v + i * 2048), idesc<BF16>(D, true), j | i);
                };
                bool ok = mbar_wait_f(&q_full, 0, &s_fail, limit) && full_wait(0);
                uint32_t committed = 0;  // bit w: o_full[w] will be raised
                if (ok) {
                    fence_after();
                    qk(0, 0);
                    commit(&s_full[0]);
                    if (n1) {
                        qk(1, 0);
                        commit(&s_full[1]);
                    }
                    commit(&kv_empty[0]);
                }
                for (uint32_t j = 0; j < n && ok; ++j) {
#pragma unroll
                    for (uint32_t w = 0; w < 2; ++w) {
                        const uint32_t mine = w ? n1 : n0;
                        if (j >= mine || !ok) continue;
                        const bool last_user = w == 1 || j >= n1, last_k_user = w == 1 || j + 1 >= n1;
                        ok = mbar_wait_f(&p_full[w], j & 1, &s_fail, limit) &&
                             (j >= n0 - 1 ? mbar_wait_f(&v_clean[j - (n0 - 1)], 0, &s_fail, limit) : full_wait(2 * j + 1));
                        if (!ok) break;
                        fence_after();
                        pv(w, j);
                        if (last_user) commit(&kv_empty[(2 * j + 1) % kStages]);
                        if (j + 1 < mine) {
                            ok = full_wait(2 * j + 2);
                            if (!ok) break;
                            fence_after();
                            qk(w, j + 1);
                            commit(&s_full[w]);
                            if (last_k_user) commit(&kv_empty[(2 * j + 2) % kStages]);
                        } else {
                            commit(&o_full[w]);
                            committed |= 1u << w;
                        }
                    }
                }
                // every product complete before TMEM and the tiles are released
                if (!ok) {
                    commit(&o_full[committed & 1]);  // one more phase of a barrier nobody waits for any more
                    mbar_drain(&o_full[committed & 1], 0);
                } else {
                    mbar_drain(&o_full[0], 0);
                    if (n1) mbar_drain(&o_full[1], 0);
                }
            }
        } else if (warp == 9) {
            // ---- loads: one thread -----------------------------------------------------------------------------
            if (lane == 0) {
                auto bar_of = [&](uint32_t i) { return i & 1 && i / 2 >= n0 - 1 ? &v_raw[i / 2 - (n0 - 1)] : &kv_full[i % kStages]; };
                auto load = [&](uint32_t i) {
                    const CUtensorMap* map = i & 1 ? &vmap : &kmap;
                    const uint32_t dst = skv + (i % kStages) * kTile;
                    uint64_t* bar = bar_of(i);
                    expect_tx(bar, kTile);
#pragma unroll
                    for (uint32_t h = 0; h < kHalves; ++h)
                        tma_tile(dst + h * kPkTileBytes, map, h, kvh, begin + (i / 2) * 128, bar);
                };
                const uint32_t q_tiles = n1 ? 2 : 1;
                expect_tx(&q_full, q_tiles * kTile);
                for (uint32_t t = 0; t < q_tiles; ++t)
#pragma unroll
                    for (uint32_t h = 0; h < kHalves; ++h)
                        tma_tile(sq + t * kTile + h * kPkTileBytes, &qmap, h, head, begin + first_row + t * 128, &q_full);
                uint32_t sent = 0;
                for (uint32_t i = 0; i < 2 * n; ++i) {
                    if (i >= kStages && !mbar_wait_f(&kv_empty[i % kStages], ((i / kStages) - 1) & 1, &s_fail, limit)) break;
                    load(i);
                    sent = i + 1;
                }
                mbar_drain(&q_full, 0);
                for (uint32_t i = sent > kStages ? sent - kStages : 0; i < sent; ++i)
                    mbar_drain(bar_of(i), i & 1 && i / 2 >= n0 - 1 ? 0 : (i / kStages) & 1);
            }
        } else {
            // ---- V tiles that some row sees only in part: elements that are not finite become 0 ---------------
            const uint32_t at = tid - 320;
            for (uint32_t j = n0 - 1; j < n; ++j) {
                if (!mbar_wait_f(&v_raw[j - (n0 - 1)], 0, &s_fail, limit)) break;
                const uint32_t v = skv + ((2 * j + 1) % kStages) * kTile;
                bool foul = false;
                for (uint32_t i = at; i < kTile / 16; i += 64) {
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
                        foul = true;
                    }
                }
                if (foul) s_foul = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&v_clean[j - (n0 - 1)]);
            }
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
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
    const dim3 grid(a.tokens / 256 + a.seqs, a.heads);
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
    if (tokens > (1u << 30) || seqs > (1u << 24)) return fail(ENX_ERR_RANGE, "enx_attn_packed: at most 2^30 tokens and 2^24 prompts");
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
