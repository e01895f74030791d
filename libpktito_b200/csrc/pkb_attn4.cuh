// The attention over a 4-bit cache: what its kernels share (the call's
// arguments, the products of one unit, the online softmax).
#pragma once

#include "pkb_cache4.cuh"
#include "pkb_device.cuh"

namespace pkb {

// The parts of an item that shares first .. last have, and its entry's rows;
// NONE where one share has it whole, it sees no tokens or there is none.
struct alignas(16) Attn4Join {
    uint32_t first, last, r0, rows;
    static constexpr uint32_t NONE = 0xFFFFFFFFu;
};

struct Attn4Args {
    Cache4 c;
    const void* q;
    void* o;
    size_t qs, os;
    const int32_t *seqs, *starts;
    uint32_t* err;
    uint32_t layer, n, rows, H, G;  // G: query heads a cached head
    uint32_t max_rows, max_blocks;  // of an entry: rows, and blocks of rows
    uint32_t team, teams;           // cached heads that go together, and how many times that (`team` times `teams` covers them)
    float scale;                    // times log2 e
    uint32_t causal, window;
    uint32_t vec, vec_o;            // q's and o's rows are 16-byte aligned
    long long timeout;
    Attn4Join* joins;               // of each item: [n][teams][max_blocks][team]
    float* part;                    // partial results, two a share and head of its team
    uint32_t max_shares;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// an 8 x 8 tile of 16-bit values, transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// two floats rounded to bf16, lo in the low half
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// x as PARTS bf16 numbers that add up to it: to its 8 first bits, or (2, 3
// parts) to all of an f16's 11 and a float's 24. Each remainder is exact.
template <int PARTS>
__device__ __forceinline__ void bf16_parts(float lo, float hi, uint32_t (&r)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
        r[i] = bf16_pair(lo, hi);
        if (i + 1 < PARTS) {
            lo = __fsub_rn(lo, __uint_as_float(r[i] << 16));
            hi = __fsub_rn(hi, __uint_as_float(r[i] & 0xFFFF0000u));
        }
    }
}

// x as PARTS f16 numbers that add up to it: to 11 and to 23 bits.
template <int PARTS>
__device__ __forceinline__ void f16_parts(float lo, float hi, uint32_t (&r)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
        const __half2 h = __floats2half2_rn(lo, hi);
        r[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (i + 1 < PARTS) {
            lo = __fsub_rn(lo, __low2float(h));
            hi = __fsub_rn(hi, __high2float(h));
        }
    }
}

// The codes of a word as f16 pairs of the whole numbers c, without the scale
// (the known way from a few bits to a float without a conversion: they become low
// bits of a number whose exponent is known, which is then subtracted):
// the nibbles in place in the mantissa of 1024 (pairs 0 and 2) and of 64
// (pairs 1 and 3), so that a word takes one shift, four ANDs and four sums.
template <int J>
__device__ __forceinline__ uint32_t c4_whole(uint32_t w) {
    const uint32_t at = J < 2 ? w : w >> 8;
    uint32_t r;
    if constexpr (J % 2 == 0) {
        asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(r) : "r"(at));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0xE408E408u));  // -1032
    } else {
        asm("lop3.b32 %0, %1, 0x00F000F0, 0x54005400, 0xEA;" : "=r"(r) : "r"(at));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0xD480D480u));  // -72
    }
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A warp's wait: every lane gives up if one does.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, long long limit) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort, limit));
}

constexpr float NEG_INF = -__builtin_huge_valf();

// e^x / e^m for partial sums: 1 where both are -inf (nothing seen yet)
__device__ __forceinline__ float rescale(float from, float to) { return from == to ? 1.0f : exp2_fast(__fsub_rn(from, to)); }

// What it costs to begin and end an item, in tiles: shares are of equal
// cost, not of equal tiles. An item is START places of no work, then its
// tiles (200 streams of 250 tokens, 4 f16 rows each: 24.4 us with none, 23.5 with two, 25.0
// with four; 64 sequences of up to 4,099: 55.2, 54.7, 55.8).
constexpr uint32_t START = 2;

// One entry's rows and tokens, and of what its rows can see the first unit,
// how many, and the places (START and the tiles, 0 where nothing is seen).
// Positions fit an int: a cache's sequences are below 2^30 tokens, and a
// window that reaches past one is none.
struct Entry {
    uint32_t seq, r0, rows, len, unit0, units, places;
    template <int NT>
    __device__ __forceinline__ uint32_t blocks(const Attn4Args& a) const { return (rows * a.G + 8 * NT - 1) / (8 * NT); }
    __device__ __forceinline__ int32_t position(uint32_t tok) const { return static_cast<int32_t>(len - rows + tok); }
};

// The first key that a row at `pos` (below 0 before the first token) sees.
__device__ __forceinline__ int32_t window_begin(const Attn4Args& a, int32_t pos) {
    const int32_t window = static_cast<int32_t>(a.window);
    return window && pos >= window ? pos - window + 1 : 0;
}

__device__ __forceinline__ Entry load_entry(const Attn4Args& a, uint32_t i) {
    Entry e;
    e.rows = c4_rows(a.c, a.seqs, a.starts, i, a.rows, &e.seq, &e.r0, a.err);
    if (e.rows > a.max_rows) {
        atomicOr(a.err, PKB_DEVERR_ARGS);
        e.rows = 0;
    }
    e.len = e.rows ? c4_len(a.c, e.seq, a.err) : 0;
    // the first row's window begins furthest back; the last row's causal end is len
    e.unit0 = static_cast<uint32_t>(window_begin(a, e.position(0))) / C4_UNIT;
    e.units = (e.len + C4_UNIT - 1) / C4_UNIT - e.unit0;
    e.places = e.len ? START + (e.units + 1) / 2 : 0;
    return e;
}

// The keys [lo, hi) that the row of an entry's token sees.
struct Keys {
    int32_t lo, hi;
};
__device__ __forceinline__ Keys keys_of(const Attn4Args& a, const Entry& e, uint32_t tok) {
    const int32_t pos = e.position(tok), len = static_cast<int32_t>(e.len);
    return {window_begin(a, pos), a.causal ? max(min(pos + 1, len), 0) : len};
}

// Many bf16 rows on the fifth-generation tensor cores (pkb_attn4_tc.cu): whether
// it takes a call, its set-up, and its launch.
bool attention4_tc_takes(const Attn4Args& a, int type);
cudaError_t prepare_attention4_tc();
cudaError_t launch_attention4_tc(const Attn4Args& a, cudaStream_t stream);

}  // namespace pkb
