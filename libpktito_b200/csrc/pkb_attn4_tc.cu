// Attention over a cache held in 4 bits, many bf16 rows (prompts), on the
// fifth-generation tensor cores.
//
// A block takes 256 rows (tokens times the query heads of one cached head) as
// two tiles of 128 and goes over its keys 64 at a time:
//     S = Q K^T   (tcgen05, Q and K from shared memory, S in TMEM)
//     P = 2^(scale log2e S - m), row sums l, a row a thread
//     O += P V    (tcgen05, P from TMEM, where it takes S's place, V from shared memory)
// Each tile has two places for S, so that the next scores lie there when a
// softmax ends, and the products of one half step run beside the softmax of
// the next. With O of both tiles that is all of TMEM. Products of 128 keys at a
// time, which have one place a tile, wait for the softmax and it for them:
// 1.18 ms against 1.09 for two prompts of 8,191 tokens, 8 heads of 128 with 4
// query heads each. They take 1.06 ms now (1,037 TFLOP/s, of the 1,662 that a library's
// bf16 product reaches; leaving out the powers of two changes 1%), and 1.17 where
// calls follow one another for so long that the power cap brings the clock
// from 1,965 to 1,770 MHz.
//
// What bounds it: the products alone take 0.94 ms. Q's 4 KB are read anew for
// every 64 keys x 16, as many cycles as the product of 128 keys takes; the
// codes' warps and the softmax, which end in 0.70 and some 0.9 ms without
// them, get in each other's way for the rest.
//
// Eight warps turn K's and V's codes into bf16, quarters of the values that they
// stand for (exactly: pkb_cache4.cuh) in the 128-byte swizzled tiles that the tensor
// cores read: K as [keys][dk], V as [dk][keys], which is how a lane's codes
// lie in the cache, in stores without bank conflicts. They load the codes a
// step of 128 keys ahead into registers: with the bf16 tiles of two steps and
// Q, shared memory has no room for a ring that covers a load's latency (1.37
// ms with one of 96 keys' codes, 1.25 so). Sixteen warps, K's and V's apart, are
// slower (1.16 ms against 1.09). One warp issues the products, eight have the
// rows; sixteen, half a row a thread, were no faster.
//
// The maximum of a row is raised only where a score passes it by 8 (a factor
// of 2^8, far inside a float), so O is rescaled in few steps.
//
// P is rounded to bf16, 8 bits: both operands of a product have one type, and
// V's values are bf16 numbers over all of its range. That is the one rounding
// here besides o's: of the result it makes 2.1e-3 (two prompts of 8,191 tokens,
// against 64 bits) where weights in float make 1.6e-3, all of which is o's. The
// few rows' kernel has a second part for the other 8 bits (pkb_attn4.cu);
// here it would double the products with V, a third of the 0.94 ms that the
// products take, and the weights' registers, which there are none of. l sums
// the weights before that rounding, in float.

#include <climits>

#include "pkb_attn4.cuh"
#include "pkb_internal.h"

namespace pkb {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int SOFT_WARPS = 8, CODE_WARPS = 8, MMA_WARP = SOFT_WARPS + CODE_WARPS;
constexpr int THREADS = 640;    // five warpgroups; the last one's three spare warps wait for the end
// A thread's registers: 96 at launch (61,440 of the SM's 65,536), then the
// rows' warps take what the others leave: 256 x 136 + 256 x 80 + 128 x 40 =
// 60,416.
constexpr int SOFT_REGS = 136, CODE_REGS = 80, ISSUE_REGS = 40;
constexpr int ROWS = 256;       // of a block, two tiles of 128
constexpr int KEYS = 128;       // of a step of K and V
constexpr int HALF = 64;        // of a product
constexpr int KV_STAGES = 2;    // steps of K and of V as bf16
constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;  // S (and P) of two halves of each tile from 0 on, O at 256 and 384

template <int NB> constexpr int slabs() { return (NB + 1) / 2; }             // of 64 dimensions, 128 rows of 128 bytes each
template <int NB> constexpr int row_tile() { return slabs<NB>() * 16384; }    // 128 rows of Q or of K
template <int NB> constexpr int v_tile() { return NB * 32 * 256; }            // dk rows of 128 keys, two slabs of 64 keys
template <int NB> constexpr int smem_bytes() {
    return 2 * row_tile<NB>() + KV_STAGES * (row_tile<NB>() + v_tile<NB>()) + 1024;
}

struct Bars {
    uint64_t k_full[KV_STAGES], k_empty[KV_STAGES], v_full[KV_STAGES], v_empty[KV_STAGES];
    uint64_t s_full[2][2], p_full[2][2], o_full[2][2], drain;  // of each tile and parity of its half steps
};

// One lane of a converged warp. The issuing warp runs its loop as a whole
// and only the products and commits are this lane's: what they take then
// stays in uniform registers (1.42 -> 1.25 ms for two prompts of 8,191
// tokens, a single thread's loop against this one).
__device__ __forceinline__ uint32_t elected() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(is));
    return is;
}

// D[tmem] (+)= A B[smem]^T, a K step of 16: A in shared memory (a descriptor) or in TMEM
__device__ __forceinline__ void mma_ss(uint32_t me, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t me, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t me, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(me)
        : "memory");
}

// 16 registers into 16 consecutive TMEM columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_st_x16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// byte offset of a 16-byte chunk of a row in a slab of 128-byte swizzled rows
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// N words of memory, as wide as they lie
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// A lane's codes and scales of a unit's K: keys g and g + 8
template <int NB>
struct KCodes {
    uint32_t w[2][NB], s[2][(NB + 1) / 2];
    __device__ __forceinline__ void load(const uint8_t* unit) {
        const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            load_words<NB>(unit + ((g + 8 * r) * 4 + t) * NB * 4, w[r]);
            const uint8_t* at = unit + 16 * 32 * NB + (g + 8 * r) * NB * 2;
            if constexpr (NB % 2 == 0) {
                load_words<NB / 2>(at, s[r]);
            } else {
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    s[r][b / 2] = reinterpret_cast<const uint16_t*>(at)[b];
                    if (b + 1 < NB) s[r][b / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[b + 1]) << 16;
                }
            }
        }
    }
    // Into 16 rows of a tile from `rows` on: eight values of a block are a
    // 16-byte chunk. Lanes of odd g take a pair of blocks the other way
    // round, so that the eight lanes of a store's quarter meet eight
    // different banks.
    __device__ __forceinline__ void store(uint8_t* rows) const {
        constexpr int PAIRED = NB / 2 * 2;
        const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3, odd = g & 1;
        uint8_t* const first_at = rows + g * 128 + (((4 * odd + t) ^ g) << 4);         // of the pair's block taken first
        uint8_t* const second_at = rows + g * 128 + (((4 * (odd ^ 1) + t) ^ g) << 4);  // and second
        uint8_t* const last_at = rows + g * 128 + ((t ^ g) << 4);                      // of a block without a pair
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const bool pair = b < PAIRED;
                const uint32_t x = pair && odd ? w[r][pair ? b ^ 1 : b] : w[r][b];
                // the block's scale in both halves: the low or the high one of its pair's word
                const uint32_t s2 = __byte_perm(s[r][b / 2], 0, pair && odd ? (b % 2 ? 0x1010 : 0x3232) : (b % 2 ? 0x3232 : 0x1010)), ms = c4_m6(s2);
                const uint4 v = make_uint4(c4_quarter<0>(x, s2, ms), c4_quarter<1>(x, s2, ms), c4_quarter<2>(x, s2, ms), c4_quarter<3>(x, s2, ms));
                *reinterpret_cast<uint4*>((!pair ? last_at : b % 2 ? second_at : first_at) + b / 2 * 16384 + r * 1024) = v;
            }
    }
};

// The same of its V: dimensions g, g + 8, .. of keys 2t, 2t + 1, 8 + 2t, 9 + 2t
template <int NB>
struct VCodes {
    uint2 w[NB];
    uint32_t s[NB][2];
    __device__ __forceinline__ void load(const uint8_t* unit) {
        constexpr int DK = NB * 32;
        const uint32_t lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            w[b] = *reinterpret_cast<const uint2*>(unit + 8 * DK + (b * 32 + lane) * 8);
#pragma unroll
            for (int c = 0; c < 2; c++) s[b][c] = *reinterpret_cast<const uint32_t*>(unit + 17 * DK + (b * C4_UNIT + 8 * c + 2 * t) * 2);
        }
    }
    // Into 16 columns of a slab of 64 keys (quarter 0 .. 3 of it). Keys from
    // `left` on become zeros: what lies there may be anything.
    __device__ __forceinline__ void store(uint8_t* slab, uint32_t quarter, int32_t left) const {
        const uint32_t lane = threadIdx.x & 31, t = lane & 3, row = lane & 7;
        // the row of a store's four 8 x 8 tiles that this lane names: dimensions from 0 and 8 on of keys 0 .. 7, then of 8 .. 15
        const uint32_t at = smem_u32(slab) + (row + (lane & 8)) * 128 + (((2 * quarter + lane / 16) ^ row) << 4);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t s2[2], ms[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                s2[c] = s[b][c];
                if (left < C4_UNIT) {
                    const int32_t key = 8 * c + 2 * static_cast<int32_t>(t);
                    if (key >= left) s2[c] = 0;
                    else if (key + 1 >= left) s2[c] &= 0xFFFFu;
                }
                ms[c] = c4_m6(s2[c]);
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t x = j ? w[b].y : w[b].x;
                asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at + (32 * b + 16 * j) * 128),
                             "r"(c4_quarter<0>(x, s2[0], ms[0])), "r"(c4_quarter<1>(x, s2[0], ms[0])), "r"(c4_quarter<2>(x, s2[1], ms[1])),
                             "r"(c4_quarter<3>(x, s2[1], ms[1]))
                             : "memory");
            }
        }
    }
};

// The largest of three
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// P of 32 columns: 2^(s scale + minus), its sum into two running ones, rounded
// to bf16, and the largest score beside it. Columns from `end` on (MASK 1, 2) and those before `first` (2) are 0.
template <int MASK>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], uint64_t scale2, uint64_t minus2, int32_t first, int32_t end, uint64_t (&sum)[2],
                                        uint32_t (&z)[16], float& top) {
#pragma unroll
    for (int x = 0; x < 16; x++) {
        float p0, p1, s0 = __uint_as_float(s[2 * x]), s1 = __uint_as_float(s[2 * x + 1]);
        if constexpr (MASK >= 1) s0 = 2 * x < end ? s0 : NEG_INF, s1 = 2 * x + 1 < end ? s1 : NEG_INF;
        if constexpr (MASK == 2) s0 = 2 * x >= first ? s0 : NEG_INF, s1 = 2 * x + 1 >= first ? s1 : NEG_INF;
        top = max3(top, s0, s1);
        unpack2(fma2_r<0>(pack2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), scale2, minus2), p0, p1);
        p0 = exp2_fast(p0);
        p1 = exp2_fast(p1);
        if constexpr (MASK >= 1) p0 = 2 * x < end ? p0 : 0.0f, p1 = 2 * x + 1 < end ? p1 : 0.0f;
        if constexpr (MASK == 2) p0 = 2 * x >= first ? p0 : 0.0f, p1 = 2 * x + 1 >= first ? p1 : 0.0f;
        sum[x & 1] = add2_rn(sum[x & 1], pack2(p0, p1));
        z[x] = bf16_pair(p0, p1);
    }
}

// The largest of 32 columns of S and `top`
template <int MASK>
__device__ __forceinline__ float largest(const uint32_t (&s)[32], int32_t first, int32_t end, float top) {
    float other = NEG_INF;
#pragma unroll
    for (int x = 0; x < 32; x += 4) {
        float v[4];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            v[y] = __uint_as_float(s[x + y]);
            if constexpr (MASK >= 1) v[y] = x + y < end ? v[y] : NEG_INF;
            if constexpr (MASK == 2) v[y] = x + y >= first ? v[y] : NEG_INF;
        }
        top = max3(top, v[0], v[1]);
        other = max3(other, v[2], v[3]);
    }
    return fmaxf(top, other);
}

// Raises a row's maximum to that of its 64 scores at s_at, and rescales its
// sum and its values, which no product is adding to.
template <int NB, int MASK>
__device__ __noinline__ void raise(uint32_t s_at, uint32_t o_at, bool begun, float scale, int32_t first, int32_t end, float& m, float& l) {
    float top = NEG_INF;
#pragma unroll 1
    for (int c = 0; c < HALF / 32; c++) {
        uint32_t a[32];
        tmem_ld_32x32b_x32(s_at + 32 * c, a);
        tmem_ld_wait(a);
        top = largest<MASK>(a, first - 32 * c, end - 32 * c, top);
    }
    const float raised = fmaxf(m, __fmul_rn(top, scale)), f = rescale(m, raised);
    m = raised;
    l *= f;
#pragma unroll 1
    for (int d = 0; begun && d < 2 * NB; d++) {
        uint32_t y[16];
        tmem_ld_32x32b_x16(o_at + 16 * d, y);
        tmem_ld_wait(y);
#pragma unroll
        for (int x = 0; x < 16; x++) y[x] = __float_as_uint(__fmul_rn(__uint_as_float(y[x]), f));
        tmem_st_x16(o_at + 16 * d, y);
    }
    tmem_st_wait();
}

// A half step of a row: its 64 scores at s_at become P in the upper half of
// their place. The weights are taken with the maximum there is, and the
// scores' own is found beside them; where that passes it by 8 (the first
// step, and few others) the maximum is raised, once the products of the half
// step before have ended (`idle`), and they are taken again.
template <int NB, int MASK, typename Idle>
__device__ __forceinline__ bool softmax_step(uint32_t s_at, uint32_t o_at, bool begun, float scale, int32_t first, int32_t end, float& m, float& l,
                                             Idle idle) {
    const uint64_t scale2 = pack2(scale, scale);
    if (!begun) raise<NB, MASK>(s_at, o_at, begun, scale, first, end, m, l);
    for (;;) {
        uint32_t a[32], b[32], z0[16], z1[16];
        const float minus = m == NEG_INF ? 0.0f : -m;
        const uint64_t minus2 = pack2(minus, minus);
        uint64_t sum[2] = {0, 0};
        tmem_ld_32x32b_x32(s_at, a);
        tmem_ld_wait(a);
        tmem_ld_32x32b_x32(s_at + 32, b);
        float top = NEG_INF;
        weights<MASK>(a, scale2, minus2, first, end, sum, z0, top);
        tmem_ld_wait(b);
        weights<MASK>(b, scale2, minus2, first - 32, end - 32, sum, z1, top);
        if (__any_sync(FULL, __fmul_rn(top, scale) > m + 8.0f)) {
            if (!idle()) return false;
            raise<NB, MASK>(s_at, o_at, begun, scale, first, end, m, l);
            continue;
        }
        tmem_st_x16(s_at + 32, z0);
        tmem_st_x16(s_at + 48, z1);
        float s0, s1, s2, s3;
        unpack2(sum[0], s0, s1);
        unpack2(sum[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        tmem_st_wait();
        return true;
    }
}

template <int REGS, bool MORE>
__device__ __forceinline__ void set_registers() {
    if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

template <int NB>
__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(Attn4Args a) {
    constexpr int DK = NB * 32;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int gave_up;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* q_tile = smem;
    uint8_t* k_tile = q_tile + 2 * row_tile<NB>();
    uint8_t* v_tiles = k_tile + KV_STAGES * row_tile<NB>();
    // the warp's index from one lane, so that the roles' branches are uniform to the compiler too
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(FULL, tid / 32, 0);
    if (tid == 0) {
        for (int i = 0; i < KV_STAGES; i++) {
            mbar_init(&bars.k_full[i], CODE_WARPS), mbar_init(&bars.v_full[i], CODE_WARPS);
            mbar_init(&bars.k_empty[i], 1), mbar_init(&bars.v_empty[i], 1);
        }
        for (int i = 0; i < 4; i++)
            mbar_init(&bars.s_full[i / 2][i % 2], 1), mbar_init(&bars.p_full[i / 2][i % 2], 4), mbar_init(&bars.o_full[i / 2][i % 2], 1);
        mbar_init(&bars.drain, 1);
        fence_mbar_init();
        gave_up = 0;
    }
    pdl_trigger();
    pdl_wait();
    // the last rows of all entries and heads, which see most, begin first
    const uint32_t rank = blockIdx.x / (a.n * a.c.heads), h = blockIdx.x % a.c.heads;
    const Entry e = load_entry(a, blockIdx.x / a.c.heads % a.n);
    const uint32_t all = e.rows * a.G, groups = (all + ROWS - 1) / ROWS;
    if (rank >= groups) return;  // the whole block
    const uint32_t group = groups - 1 - rank, row0 = group * ROWS, tiles = all - row0 > 128 ? 2 : 1;
    const uint32_t last = min(row0 + ROWS, all) - 1;
    const int32_t lo = keys_of(a, e, row0 / a.G).lo, hi = keys_of(a, e, last / a.G).hi;
    const uint32_t unit0 = static_cast<uint32_t>(lo / C4_UNIT);
    const uint32_t units = hi > lo ? static_cast<uint32_t>((hi + C4_UNIT - 1) / C4_UNIT) - unit0 : 0;
    const uint32_t steps = (units * C4_UNIT + KEYS - 1) / KEYS, halves = (units * C4_UNIT + HALF - 1) / HALF;
    const int32_t key_base = static_cast<int32_t>(unit0 * C4_UNIT);
    if (warp == MMA_WARP) {
        tmem_alloc(&tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    // Q, zeros for rows there are none of; a negative scale's sign goes with it
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    constexpr int CHUNKS = (ROWS * (DK / 8) + THREADS - 1) / THREADS;
    uint4 chunk_of[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {  // all loads before the first store
        const uint32_t x = tid + i * THREADS, chunk = x % (DK / 8), row = row0 + x / (DK / 8), tok = row / a.G;
        chunk_of[i] = make_uint4(0, 0, 0, 0);
        if (x < ROWS * (DK / 8) && row < all) {
            const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + static_cast<size_t>(e.r0 + tok) * a.qs +
                                     static_cast<size_t>(h * a.G + row - tok * a.G) * DK + 8 * chunk;
            if (a.vec) {
                chunk_of[i] = *reinterpret_cast<const uint4*>(p);
            } else {
                alignas(16) __nv_bfloat16 y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = p[j];
                chunk_of[i] = *reinterpret_cast<const uint4*>(y);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
        const uint32_t x = tid + i * THREADS, chunk = x % (DK / 8), r = x / (DK / 8);
        const uint4 v = chunk_of[i];
        if (x < ROWS * (DK / 8))
            *reinterpret_cast<uint4*>(q_tile + (r / 128) * row_tile<NB>() + (chunk / 8) * 16384 + swizzled(r % 128, chunk & 7)) =
                make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
    }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins

    // one instruction sets a warpgroup's registers, and all of its warps run it: the last one's spare warps too
    if (warp >= MMA_WARP) {
        set_registers<ISSUE_REGS, false>();
        if (warp == MMA_WARP) {
            // descriptors hold addresses in units of 16 bytes, in their low bits
            const uint64_t q_at = sw128_kmajor_desc(smem_u32(q_tile)), k_at = sw128_kmajor_desc(smem_u32(k_tile)),
                           v_at = sw128_kmajor_desc(smem_u32(v_tiles));
            constexpr uint32_t QK = bf16_instr_desc(128, HALF), PV = bf16_instr_desc(128, DK);
            const uint32_t me = elected();
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = ok && warp_wait(bar, parity, &gave_up, a.timeout);
                if (ok) tc_fence_after();
                return ok;
            };
            auto scores = [&](uint32_t t, uint32_t i) {
                const uint64_t qd = q_at + t * (row_tile<NB>() / 16), kd = k_at + i / 2 % KV_STAGES * (row_tile<NB>() / 16) + i % 2 * (HALF * 8);
                const uint32_t to = S_COL + 128 * t + HALF * (i % 2);
    #pragma unroll
                for (int k = 0; k < DK / 16; k++) mma_ss(me, to, qd + k / 4 * 1024 + k % 4 * 2, kd + k / 4 * 1024 + k % 4 * 2, QK, k > 0);
                commit(me, &bars.s_full[t][i % 2]);
                if (t + 1 == tiles && i % 2) commit(me, &bars.k_empty[i / 2 % KV_STAGES]);
            };
            auto values = [&](uint32_t t, uint32_t i) {
                const uint64_t vd = v_at + i / 2 % KV_STAGES * (v_tile<NB>() / 16) + i % 2 * (DK * 8);
                const uint32_t from = S_COL + 128 * t + HALF * (i % 2) + 32;
    #pragma unroll
                for (int k = 0; k < HALF / 16; k++) mma_ts(me, O_COL + 128 * t, from + 8 * k, vd + 2 * k, PV, i > 0 || k > 0);
                commit(me, &bars.o_full[t][i % 2]);
                if (t + 1 == tiles && i % 2) commit(me, &bars.v_empty[i / 2 % KV_STAGES]);
            };
            if (halves && wait(&bars.k_full[0], 0)) {
                for (uint32_t i = 0; i < halves && i < 2; i++)
                    for (uint32_t t = 0; t < tiles; t++) scores(t, i);
            }
            // a tile's scores of the half step after next follow its values: they
            // take P's place in TMEM, and products of one thread run in their order
            for (uint32_t i = 0; ok && i < halves; i++) {
                const uint32_t j = i / 2, st = j % KV_STAGES, ph = j / KV_STAGES & 1, st1 = (j + 1) % KV_STAGES, ph1 = (j + 1) / KV_STAGES & 1;
                if (i % 2 == 0 && !wait(&bars.v_full[st], ph)) break;
                for (uint32_t t = 0; t < tiles; t++) {
                    if (!wait(&bars.p_full[t][i % 2], j & 1)) break;
                    values(t, i);
                    if (i + 2 >= halves) continue;
                    if (t == 0 && i % 2 == 0 && !wait(&bars.k_full[st1], ph1)) break;
                    scores(t, i + 2);
                }
            }
            if (!ok) {
                gave_up = 1;
                if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
                // what was issued finishes before TMEM is freed
                commit(me, &bars.drain);
                if (me) mbar_drain(&bars.drain, 0, a.timeout);
                __syncwarp();
            }
        }
    } else if (warp >= SOFT_WARPS) {
        // codes to values: a warp a unit of each step
        set_registers<CODE_REGS, false>();
        const uint32_t w = warp - SOFT_WARPS, per = a.c.pshift - 4;
        const int32_t* table = a.c.table + static_cast<size_t>(e.seq) * a.c.max_pages;
        const uint8_t* head = a.c.pages + a.layer * a.c.layer_bytes + h * a.c.head_bytes;
        KCodes<NB> k;
        VCodes<NB> v;
        int32_t page = 0;  // of the step that is loaded next
        auto look = [&](uint32_t i) {
            const uint32_t u = 8 * i + w;
            page = u < units ? table[(unit0 + u) >> per] : 0;
        };
        // where a unit lies; past the last one any codes will do, they become zeros or are hidden
        auto unit_at = [&](uint32_t i) {
            uint32_t p = static_cast<uint32_t>(page);
            if (p >= a.c.n_pages) {
                if (lane == 0) atomicOr(a.err, PKB_DEVERR_ARGS);  // any page will do, the rows are not defined
                p = 0;
            }
            return head + p * a.c.page_bytes + ((unit0 + 8 * i + w) & ((1u << per) - 1)) * (18 * DK);
        };
        const uint8_t* at = nullptr;
        if (steps) {
            look(0);
            at = unit_at(0);
            k.load(at);
            v.load(at);
            look(1);
        }
        for (uint32_t i = 0; i < steps; i++) {
            const uint32_t st = i % KV_STAGES, ph = i / KV_STAGES & 1;
            const bool more = i + 1 < steps;
            bool ok = warp_wait(&bars.k_empty[st], ph ^ 1, &gave_up, a.timeout);
            if (ok) {
                k.store(k_tile + st * row_tile<NB>() + 16 * w * 128);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.k_full[st]);
                if (more) {
                    at = unit_at(i + 1);
                    k.load(at);
                    look(i + 2);
                }
                ok = warp_wait(&bars.v_empty[st], ph ^ 1, &gave_up, a.timeout);
            }
            if (ok) {
                v.store(v_tiles + st * v_tile<NB>() + w / 4 * (DK * 128), w % 4, hi - key_base - static_cast<int32_t>(i * KEYS + 16 * w));
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.v_full[st]);
                if (more) v.load(at);
            }
            if (!ok) {
                gave_up = 1;
                if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
                break;
            }
        }
    } else if (warp / 4 < tiles) {
        // the rows: thread i of a tile's four warps has row i
        set_registers<SOFT_REGS, true>();
        const uint32_t t = warp / 4, row = row0 + tid, tok = row / a.G;
        const Keys span = keys_of(a, e, min(tok, e.rows - 1));  // rows there are none of see what the last one does
        const uint32_t at = tmem + ((warp % 4) * 32 << 16), s_at = at + S_COL + 128 * t, o_at = at + O_COL + 128 * t;
        const float scale = fminf(fmaxf(__fmul_rn(4.0f, fabsf(a.scale)), 0x1p-149f), 3.0e38f);  // K comes as quarters; a scale of 0 as the least there is
        float m = NEG_INF, l = 0.0f;
        bool ok = true;
        // the values up to half step i are in O
        auto values_in = [&](uint32_t i) {
            const bool in = warp_wait(&bars.o_full[t][i % 2], i / 2 & 1, &gave_up, a.timeout);
            tc_fence_after();
            return in;
        };
        for (uint32_t i = 0; i < halves; i++) {
            ok = warp_wait(&bars.s_full[t][i % 2], i / 2 & 1, &gave_up, a.timeout);
            if (!ok) break;
            tc_fence_after();
            auto idle = [&]() { return i == 0 || values_in(i - 1); };
            const uint32_t from = s_at + HALF * (i % 2);
            const int32_t key0 = key_base + static_cast<int32_t>(i * HALF), first = span.lo - key0, end = span.hi - key0;
            const bool before = __any_sync(FULL, first > 0), behind = __any_sync(FULL, end < HALF);
            if (before) ok = softmax_step<NB, 2>(from, o_at, i > 0, scale, first, end, m, l, idle);
            else if (behind) ok = softmax_step<NB, 1>(from, o_at, i > 0, scale, 0, end, m, l, idle);
            else ok = softmax_step<NB, 0>(from, o_at, i > 0, scale, 0, HALF, m, l, idle);
            if (!ok) break;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[t][i % 2]);
        }
        if (halves && ok) ok = values_in(halves - 1);
        if (!ok) {
            gave_up = 1;
            if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
        } else {
            // V came as quarters; a row that sees nothing has sum 0 and is zeros; a NaN sum gives NaNs
            const float inv = l == 0.0f ? 0.0f : __fdiv_rn(4.0f, l);
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o) + static_cast<size_t>(e.r0 + tok) * a.os +
                                 static_cast<size_t>(h * a.G + row - tok * a.G) * DK;
#pragma unroll
            for (int c = 0; c < NB; c++) {
                uint32_t y[32];
                if (steps) {
                    tmem_ld_32x32b_x32(o_at + 32 * c, y);
                    tmem_ld_wait(y);
                } else {
#pragma unroll
                    for (int x = 0; x < 32; x++) y[x] = 0;
                }
                alignas(16) uint32_t z[16];
#pragma unroll
                for (int x = 0; x < 16; x++) z[x] = bf16_pair(__fmul_rn(__uint_as_float(y[2 * x]), inv), __fmul_rn(__uint_as_float(y[2 * x + 1]), inv));
                if (row < all) {
                    if (a.vec_o) {
#pragma unroll
                        for (int x = 0; x < 4; x++) reinterpret_cast<uint4*>(out + 32 * c)[x] = make_uint4(z[4 * x], z[4 * x + 1], z[4 * x + 2], z[4 * x + 3]);
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; x++)
                            out[32 * c + x] = __ushort_as_bfloat16(static_cast<unsigned short>(x & 1 ? z[x / 2] >> 16 : z[x / 2] & 0xFFFFu));
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_slot, TMEM_COLS);
    }
}

template <int NB>
cudaError_t launch_one(const Attn4Args& a, cudaStream_t s) {
    const uint64_t grid = (static_cast<uint64_t>(a.max_rows) * a.G + ROWS - 1) / ROWS * a.c.heads * a.n;
    if (grid > INT_MAX) return cudaErrorInvalidConfiguration;
    return c4_launch(prompt_kernel<NB>, static_cast<uint32_t>(grid), THREADS, smem_bytes<NB>(), s, a);
}

}  // namespace

bool attention4_tc_takes(const Attn4Args& a, int type) { return type == PKB_BF16 && a.c.dk <= 128; }

cudaError_t prepare_attention4_tc() {
    cudaError_t e = cudaFuncSetAttribute(prompt_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<1>());
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prompt_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<2>());
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prompt_kernel<3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<3>());
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prompt_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<4>());
    return e;
}

cudaError_t launch_attention4_tc(const Attn4Args& a, cudaStream_t stream) {
    const cudaError_t e = a.c.dk == 32   ? launch_one<1>(a, stream)
                          : a.c.dk == 64 ? launch_one<2>(a, stream)
                          : a.c.dk == 96 ? launch_one<3>(a, stream)
                                         : launch_one<4>(a, stream);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace pkb
