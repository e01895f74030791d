// The cache held in 4 bits (include/pktito_b200.h, pkb_cache4): rows into its
// pages and back, and its page operations.
//
// Rows. Append reads each value once (2 or 4 bytes) and writes 4.5 bits of
// it, read does the reverse: many rows are bound by memory (24 segments'
// 28.8 M float values appended and read back: 260 MB in 61 us, 4.3 TB/s, of 40
// at the rate of a copy), few by the latency of some dependent loads
// (an entry's rows, its length, its page, the row). A warp takes one unit's K
// or V (16 tokens of one head), four lanes a token, so that a lane's eight
// values of a block are one word of K's codes. V's words mix 4 tokens: append puts
// them together from bytes in shared memory, read takes them apart with 8 x 8
// transposes in registers. A byte is one token's, so a unit that the call
// covers in part is written a byte at a time beside the tokens it leaves
// alone.
//
// Page operations. One block plans (it checks the lists, finds the lowest
// free pages by a scan of refs, and refuses before anything is changed), a
// grid applies: table rows, references and the pages' bytes. They are bound
// by the copied bytes where pages are copied (192 sessions of up to 4,001
// tokens freed, compacted and some copied: 1.07 GB each way in 0.40 ms, of 0.33 at a
// copy's rate), else by the launches and the latency of the plan's few
// dependent reads (32 hypotheses' step of free, fork and grow: 18.6 us in a
// graph, 44 from Python).

#include <climits>

#include "pkb_cache4.cuh"
#include "pkb_device.cuh"
#include "pkb_internal.h"

namespace pkb {

namespace {

constexpr int ROW_WARPS = 8;
constexpr uint32_t FULL = 0xFFFFFFFFu;

struct RowArgs {
    Cache4 c;
    const int32_t *seqs, *starts, *status;  // status: of the page operation before, or null
    uint32_t* err;
    size_t ks, vs;
    uint32_t layer, n, rows, slots;
};

// The last entry whose first row is at most row 16 x + 15: thirty-two probes
// a step, or all at once.
__device__ __forceinline__ uint32_t entry_at(const int32_t* starts, uint32_t n, uint32_t x) {
    const uint32_t lane = threadIdx.x & 31;
    if (n <= 256) {  // eight entries a lane, all asked for at once
        uint32_t below = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            const uint32_t i = j * 32 + lane;
            below += i < n && static_cast<uint32_t>(starts[i]) / C4_UNIT <= x;
        }
        below = __reduce_add_sync(FULL, below);
        return below ? below - 1 : 0;
    }
    uint32_t lo = 0, hi = n;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const bool below = i < hi && static_cast<uint32_t>(starts[i]) / C4_UNIT <= x;
        const uint32_t last = 31 - __clz(__ballot_sync(FULL, below) | 1u);
        lo += last * step;
        hi = lo + step < hi ? lo + step : hi;
    }
    return lo;
}

// Where a warp's unit lies, and which of its tokens the call has: token r is
// row `row0 + r` for r in [first, last).
struct UnitRows {
    uint8_t* bytes;
    const int32_t* users;  // of its page
    int64_t row0;
    int first, last;
};

// The unit of a slot. The first 2 n slots are the entries' first two units each
// (all there are of up to 17 rows), found without a search; the others those
// that longer entries have beside them, (rows - 2) / 16 at most, so that
// counting them from starts[i] / 16 leaves every entry room. (One row of each
// of 256 sequences appended and read: 16.4 us, 18.5 with a search for every
// slot, 14.5 with one warp for an entry's two units, whose loop costs the long
// entries 62 -> 67.)
__device__ __forceinline__ UnitRows warp_unit(const RowArgs& a, uint32_t slot, uint32_t h) {
    UnitRows u = {nullptr, nullptr, 0, 0, 0};
    uint32_t i = slot / 2, k = slot % 2;
    if (i >= a.n) {
        const uint32_t x = slot - 2 * a.n;
        i = entry_at(a.starts, a.n, x);
        const uint32_t at = static_cast<uint32_t>(a.starts[i]) / C4_UNIT;
        if (x < at) return u;
        k = 2 + x - at;
    }
    uint32_t seq, r0;
    const uint32_t rows = c4_rows(a.c, a.seqs, a.starts, i, a.rows, &seq, &r0, a.err);
    if (!rows) return u;
    const uint32_t len = c4_len(a.c, seq, a.err);
    if (rows > len) {
        if ((threadIdx.x & 31) == 0) atomicOr(a.err, PKB_DEVERR_ARGS);
        return u;
    }
    const uint32_t pos0 = len - rows, unit = pos0 / C4_UNIT + k;
    if (unit > (len - 1) / C4_UNIT) return u;  // the entry has no such unit
    u.bytes = c4_unit(a.c, a.layer, seq, h, unit, &u.users, a.err);
    const int64_t t0 = static_cast<int64_t>(unit) * C4_UNIT - pos0;
    u.row0 = r0 + t0;
    u.first = t0 < 0 ? static_cast<int>(-t0) : 0;
    u.last = static_cast<int64_t>(rows) - t0 < C4_UNIT ? static_cast<int>(rows - t0) : C4_UNIT;
    return u;
}

template <int NB> __host__ __device__ constexpr int v_row() { return NB * 16 + 8; }  // a token's V bytes, and 8 against bank conflicts

// A block's scale and its codes + 8, from four lanes' eight values each.
//
// The scale is amax times the float nearest to 1 / 7, rounded and cut to 5
// significant bits (the quotient's own, but where amax lies within a step
// below 7 s). A code is rint(x / s), ties to even: from x times an approximate
// 1 / s, whose remainder x - c s is exact in one FMA and says whether c is the
// nearest. It is not, or may be a tie, in few warps: the others skip the
// correction. No division: with a correctly rounded one a value the kernel
// took 49 us for 28.8 M float values, 32 so.
__device__ __forceinline__ float quantize_block(float (&f)[8], uint32_t (&nib)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, abs_bits(f[i]));
    m = max(m, __shfl_xor_sync(FULL, m, 1));
    m = max(m, __shfl_xor_sync(FULL, m, 2));
    const bool scaled = block_scaled(m);
    float s = __uint_as_float(__float_as_uint(__fmul_rn(__uint_as_float(m), 0.14285714924335479736f)) & 0xFFF80000u);
    if (__any_sync(FULL, !scaled)) {  // zeros, with a scale that divides
        s = scaled ? s : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = scaled ? f[i] : 0.0f;
    }
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    float left[8], worst = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // 8 + c in the low bits of 1.5 2^23 + 8 + x / s (8 is even, so ties stay ties)
        const float sum = __fadd_rn(__fmul_rn(f[i], inv), 12582920.0f);
        nib[i] = __float_as_uint(sum);
        left[i] = __fmaf_rn(__fsub_rn(12582920.0f, sum), s, f[i]);
        worst = fmaxf(worst, fabsf(left[i]));
    }
    const float half = 0.5f * s;
    if (__any_sync(FULL, worst >= half)) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (fabsf(left[i]) > half || (fabsf(left[i]) == half && (nib[i] & 1))) nib[i] += left[i] > 0.0f ? 1 : -1;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) nib[i] &= 15u;
    return scaled ? s : 0.0f;
}

// One unit's K or V; x: the head's values of row 0, xs apart. A page that
// other sequences hold too keeps its bytes: how many do is read beside the
// rows and looked at before the first store.
template <typename T, int NB, bool VEC>
__device__ __forceinline__ void append_unit(const T* x, size_t xs, const UnitRows& u, bool is_v, uint8_t* vb, uint32_t* err) {
    constexpr int DK = NB * 32;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    const int32_t users = *u.users;
    x += 8 * t;
    uint8_t* codes = u.bytes + (is_v ? 8 * DK : 0);
    __nv_bfloat16* scales = reinterpret_cast<__nv_bfloat16*>(u.bytes + (is_v ? 17 * DK : 16 * DK));
#pragma unroll
    for (int r = 0; r < 2; r++) {
        // lanes 4 g .. 4 g + 3 have token g or g + 8, eight values of each block
        const int token = static_cast<int>(g) + 8 * r;
        const bool valid = token >= u.first && token < u.last;
        if (!__any_sync(FULL, valid)) continue;
        float f[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int i = 0; i < 8; i++) f[b][i] = 0.0f;
            if (valid) c4_load8<T, VEC>(x + (u.row0 + token) * xs + b * 32, f[b]);
        }
        const bool write = valid && users == 1;
        uint32_t words[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t nib[8];
            const __nv_bfloat16 s = __float2bfloat16_rn(quantize_block(f[b], nib));  // exact: 5 bits
            if (!is_v) {
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) w |= nib[i] << (4 * (i / 2) + 16 * (i % 2));
                words[b] = w;
                if (write && t == 0) scales[token * NB + b] = s;
            } else {
                const uint32_t lo = nib[0] | nib[1] << 8 | nib[2] << 16 | nib[3] << 24;
                const uint32_t hi = nib[4] | nib[5] << 8 | nib[6] << 16 | nib[7] << 24;
                // values 8 apart share a byte: the even lane of a pair makes the first four bytes, the odd one the others
                const uint32_t got = __shfl_xor_sync(FULL, t & 1 ? lo : hi, 1);
                const uint32_t w = t & 1 ? got | hi << 4 : lo | got << 4;
                *reinterpret_cast<uint32_t*>(vb + token * v_row<NB>() + (b * 2 + t / 2) * 8 + (t & 1) * 4) = w;
                if (write && t == 0) scales[b * C4_UNIT + token] = s;
            }
        }
        if (!is_v && write) {
            uint32_t* at = reinterpret_cast<uint32_t*>(codes) + (token * 4 + t) * NB;
            if constexpr (NB % 4 == 0) {
#pragma unroll
                for (int b = 0; b < NB; b += 4) *reinterpret_cast<uint4*>(at + b) = make_uint4(words[b], words[b + 1], words[b + 2], words[b + 3]);
            } else {
#pragma unroll
                for (int b = 0; b < NB; b++) at[b] = words[b];
            }
        }
    }
    if (users != 1) {
        if (lane == 0) atomicOr(err, PKB_DEVERR_ARGS);
        return;
    }
    if (!is_v) return;
    __syncwarp();
    const uint32_t have = (0xFFFFu >> (C4_UNIT - u.last)) & (0xFFFFu << u.first);
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int wi = i * 32 + lane, blk = wi / 64, j = wi % 2;
        const uint8_t* at = vb + (blk * 2 + j) * 8 + wi / 8 % 8;
        const int pair = wi / 2 % 4;
        // byte 2 e + c of a word is token 8 c + 2 pair + e
        const uint32_t mine = have >> (2 * pair);
        if ((mine & 0x0303u) == 0) continue;
        uint8_t y[4];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int c = 0; c < 2; c++) y[2 * e + c] = at[(8 * c + 2 * pair + e) * v_row<NB>()];
        if ((mine & 0x0303u) == 0x0303u) {
            reinterpret_cast<uint32_t*>(codes)[wi] = y[0] | y[1] << 8 | y[2] << 16 | static_cast<uint32_t>(y[3]) << 24;
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    if (mine >> (8 * c + e) & 1) codes[4 * wi + 2 * e + c] = y[2 * e + c];
        }
    }
}

// A warp's slot, head, and whether its V: K's and V's warps of a unit are neighbours
struct RowItem {
    size_t slot;
    uint32_t h;
    bool is_v;
    __device__ __forceinline__ explicit RowItem(const RowArgs& a) {
        const size_t item = static_cast<size_t>(blockIdx.x) * ROW_WARPS + threadIdx.x / 32;
        is_v = item & 1;
        h = static_cast<uint32_t>((item >> 1) % a.c.heads);
        slot = (item >> 1) / a.c.heads;
    }
};

template <typename T, int NB, bool VEC>
__global__ void __launch_bounds__(ROW_WARPS * 32, NB == 8 ? 2 : 4) append_kernel(const T* k, const T* v, RowArgs a) {
    __shared__ alignas(16) uint8_t stage[ROW_WARPS][C4_UNIT * v_row<NB>()];
    pdl_trigger();
    pdl_wait();
    if (a.status && *a.status) return;  // the tokens that the rows are for were not taken
    const RowItem me(a);
    if (me.slot >= a.slots) return;
    const UnitRows u = warp_unit(a, static_cast<uint32_t>(me.slot), me.h);
    if (u.bytes)
        append_unit<T, NB, VEC>((me.is_v ? v : k) + me.h * (NB * 32), me.is_v ? a.vs : a.ks, u, me.is_v, stage[threadIdx.x / 32], a.err);
}

// a bf16 pair's two values at p (8-byte, or 4-byte aligned for 16-bit types, where VEC)
template <typename T, bool VEC>
__device__ __forceinline__ void store_pair(T* p, uint32_t pair) {
    const float lo = __uint_as_float(pair << 16), hi = __uint_as_float(pair & 0xFFFF0000u);
    if constexpr (!VEC) {
        p[0] = c4_round<T>(lo);
        p[1] = c4_round<T>(hi);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(p) = make_float2(lo, hi);
    } else {
        alignas(4) T y[2] = {c4_round<T>(lo), c4_round<T>(hi)};
        *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(y);
    }
}

// One unit's K or V, to the head's values of row 0, xs apart
template <typename T, int NB, bool VEC>
__device__ __forceinline__ void read_unit(T* x, size_t xs, const UnitRows& u, bool is_v) {
    constexpr int DK = NB * 32;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    if (!is_v) {
        // a lane's words of tokens g and g + 8: eight values of each block
        uint32_t w[2][NB];
        uint16_t s[2][NB];
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                w[r][b] = reinterpret_cast<const uint32_t*>(u.bytes)[((g + 8 * r) * 4 + t) * NB + b];
                s[r][b] = reinterpret_cast<const uint16_t*>(u.bytes + 16 * DK)[(g + 8 * r) * NB + b];
            }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int token = static_cast<int>(g) + 8 * r;
            if (token < u.first || token >= u.last) continue;
            T* to = x + (u.row0 + token) * xs + 8 * t;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t s2 = s[r][b] | static_cast<uint32_t>(s[r][b]) << 16;
                const uint32_t p[4] = {c4_whole_pair<0>(w[r][b], s2), c4_whole_pair<1>(w[r][b], s2), c4_whole_pair<2>(w[r][b], s2), c4_whole_pair<3>(w[r][b], s2)};
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    f[2 * i] = __uint_as_float(p[i] << 16);
                    f[2 * i + 1] = __uint_as_float(p[i] & 0xFFFF0000u);
                }
                c4_store8<T, VEC>(to + b * 32, f);
            }
        }
        return;
    }
    // A lane's words have pairs of tokens of dimensions g, g + 8, ..: eight by
    // eight transposes make them pairs of dimensions of token g
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const uint2 w = *reinterpret_cast<const uint2*>(u.bytes + 8 * DK + (b * 32 + lane) * 8);
        uint32_t s2[2];
#pragma unroll
        for (int c = 0; c < 2; c++) s2[c] = *reinterpret_cast<const uint32_t*>(u.bytes + 17 * DK + (b * C4_UNIT + 8 * c + 2 * t) * 2);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t y = j ? w.y : w.x;
            uint32_t p[2][2] = {{c4_whole_pair<0>(y, s2[0]), c4_whole_pair<1>(y, s2[0])}, {c4_whole_pair<2>(y, s2[1]), c4_whole_pair<3>(y, s2[1])}};
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int token = static_cast<int>(g) + 8 * c;
                const bool valid = token >= u.first && token < u.last;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    uint32_t pair;
                    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pair) : "r"(p[c][r]));
                    if (valid) store_pair<T, VEC>(x + (u.row0 + token) * xs + 32 * b + 16 * j + 8 * r + 2 * t, pair);
                }
            }
        }
    }
}

template <typename T, int NB, bool VEC>
__global__ void __launch_bounds__(ROW_WARPS * 32, NB == 8 ? 5 : 8) read_kernel(T* k, T* v, RowArgs a) {
    pdl_trigger();
    pdl_wait();
    const RowItem me(a);
    if (me.slot >= a.slots) return;
    const UnitRows u = warp_unit(a, static_cast<uint32_t>(me.slot), me.h);
    if (u.bytes) read_unit<T, NB, VEC>((me.is_v ? v : k) + me.h * (NB * 32), me.is_v ? a.vs : a.ks, u, me.is_v);
}

// ------------------------------------------------------------ page operations --

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_REFS = 16;  // refs a thread looks at a step
constexpr uint32_t COPY_CHUNK = 16384;

enum { OP_GROW = 0, OP_FORK = 1, OP_COPY = 2, OP_FREE = 3 };

// The work area: counts, then a mark a sequence, each entry's first new
// page, the free pages taken, and the pages to copy from and to. compact
// uses the last three for the holes, the pages that move and where to.
struct PlanWork {
    uint32_t* count;  // [0] new pages (compact: pages that move), [1] used pages
    uint32_t *mark, *first, *page, *from, *to;
};

struct PlanArgs {
    Cache4 c, src;  // src: copy's other cache (else c)
    const int32_t *a, *b, *num;  // sequences (the ones read first), added or taken tokens
    uint32_t n;
    int op;
    int32_t* status;
    PlanWork w;
};

// The sum of x over the threads before this one, and over all in *total.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* total, T* buf) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    T s = x;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const T y = __shfl_up_sync(FULL, s, d);
        if (lane >= d) s += y;
    }
    if (lane == 31) buf[warp] = s;
    __syncthreads();
    if (warp == 0) {
        T z = buf[lane];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const T y = __shfl_up_sync(FULL, z, d);
            if (lane >= d) z += y;
        }
        buf[lane] = z;
    }
    __syncthreads();
    *total = buf[31];
    const T before = (warp ? buf[warp - 1] : 0) + s - x;
    __syncthreads();
    return before;
}

__device__ __forceinline__ uint32_t pages_of(const Cache4& c, uint32_t tokens) {
    return static_cast<uint32_t>((static_cast<uint64_t>(tokens) + (1u << c.pshift) - 1) >> c.pshift);
}

// Entry i's new pages, and what is wrong with it.
__device__ __forceinline__ uint32_t plan_entry(const PlanArgs& p, uint32_t i, int* bad) {
    const int32_t* changed = p.op == OP_FORK || p.op == OP_COPY ? p.b : p.a;
    const int32_t s = changed[i];
    if (s < 0 || static_cast<uint32_t>(s) >= p.c.max_seqs) {
        *bad = PKB_CACHE4_BAD;
        return 0;
    }
    p.w.mark[s] = i;
    if (p.op == OP_FREE) return 0;
    const int32_t num = p.num[i], len = p.c.lens[s];
    const uint64_t room = static_cast<uint64_t>(p.c.max_pages) << p.c.pshift;
    if (num < 0 || len < 0) {
        *bad = PKB_CACHE4_BAD;
        return 0;
    }
    if (p.op == OP_GROW) {
        const uint64_t after = static_cast<uint64_t>(len) + num;
        if (after > room || after > INT_MAX) {
            *bad = max(*bad, static_cast<int>(PKB_CACHE4_LONG));
            return 0;
        }
        return pages_of(p.c, static_cast<uint32_t>(after)) - pages_of(p.c, len);
    }
    const int32_t r = p.a[i];
    if (len != 0 || r < 0 || static_cast<uint32_t>(r) >= p.src.max_seqs || num > p.src.lens[r]) {
        *bad = PKB_CACHE4_BAD;
        return 0;
    }
    if (static_cast<uint64_t>(num) > room || static_cast<uint64_t>(num) > static_cast<uint64_t>(p.src.max_pages) << p.src.pshift) {
        *bad = max(*bad, static_cast<int>(PKB_CACHE4_LONG));
        return 0;
    }
    return p.op == OP_COPY ? pages_of(p.c, num) : (num & ((1u << p.c.pshift) - 1)) != 0;
}

__device__ __forceinline__ uint32_t entry_of(const uint32_t* first, uint32_t n, uint32_t j) {
    uint32_t lo = 0, hi = n;  // the last i with first[i] <= j
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= j) lo = mid; else hi = mid;
    }
    return lo;
}

// The 16 refs of a thread's step at p0, those past the end as used.
__device__ __forceinline__ void load_refs(const Cache4& c, uint32_t p0, int32_t (&r)[PLAN_REFS]) {
    if (p0 + PLAN_REFS <= c.n_pages && (reinterpret_cast<uintptr_t>(c.refs) & 15) == 0) {
#pragma unroll
        for (int q = 0; q < PLAN_REFS / 4; q++) {
            const int4 v = reinterpret_cast<const int4*>(c.refs + p0)[q];
            r[4 * q] = v.x, r[4 * q + 1] = v.y, r[4 * q + 2] = v.z, r[4 * q + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < PLAN_REFS; q++) r[q] = p0 + q < c.n_pages ? c.refs[p0 + q] : 1;
    }
}

// free's part for entry i: its pages lose a user, its row is emptied.
__device__ __forceinline__ void free_place(const PlanArgs& p, uint32_t i, uint32_t j, uint32_t* err) {
    int32_t* at = p.c.table + static_cast<size_t>(p.a[i]) * p.c.max_pages + j;
    const int32_t page = *at;
    if (page >= 0) {
        if (static_cast<uint32_t>(page) < p.c.n_pages) atomicSub(p.c.refs + page, 1);
        else atomicOr(err, PKB_DEVERR_ARGS);
        *at = -1;
    }
    if (j == 0) p.c.lens[p.a[i]] = 0;
}

// alone: free, all of it in this block
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(PlanArgs p, bool alone, uint32_t* err) {
    __shared__ uint32_t buf[32];
    __shared__ uint64_t wide[32];
    __shared__ int worst;
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x;
    if (tid == 0) worst = 0;
    __syncthreads();
    int bad = 0;
    uint64_t wanted = 0;  // a sum of wishes, which may pass 32 bits
    for (uint32_t i0 = 0; i0 < p.n; i0 += PLAN_THREADS) {
        const uint32_t i = i0 + tid;
        const uint64_t need = i < p.n ? plan_entry(p, i, &bad) : 0;
        uint64_t sum;
        const uint64_t before = block_scan(need, &sum, wide);
        if (i < p.n) p.w.first[i] = static_cast<uint32_t>(wanted + before);
        wanted += sum;
    }
    if (wanted > p.c.n_pages) bad = max(bad, static_cast<int>(PKB_CACHE4_FULL));
    const uint32_t total = static_cast<uint32_t>(wanted);
    __syncthreads();
    // a sequence listed twice has one of its entries' marks
    const int32_t* changed = p.op == OP_FORK || p.op == OP_COPY ? p.b : p.a;
    for (uint32_t i = tid; i < p.n; i += PLAN_THREADS) {
        const int32_t s = changed[i];
        if (s >= 0 && static_cast<uint32_t>(s) < p.c.max_seqs && p.w.mark[s] != i) bad = PKB_CACHE4_BAD;
    }
    if (bad) atomicMax(&worst, bad);
    __syncthreads();
    uint32_t found = 0;
    if (!worst) {
        for (uint32_t q0 = 0; q0 < p.c.n_pages && found < total; q0 += PLAN_THREADS * PLAN_REFS) {
            const uint32_t p0 = q0 + tid * PLAN_REFS;
            int32_t r[PLAN_REFS];
            load_refs(p.c, p0, r);
            uint32_t mine = 0;
#pragma unroll
            for (int q = 0; q < PLAN_REFS; q++) mine += r[q] == 0;
            uint32_t sum;
            uint32_t at = found + block_scan(mine, &sum, buf);
#pragma unroll
            for (int q = 0; q < PLAN_REFS; q++)
                if (r[q] == 0 && at < total) p.w.page[at++] = p0 + q;
            found += sum;
        }
    }
    const int status = worst ? worst : found < total ? static_cast<int>(PKB_CACHE4_FULL) : 0;
    if (tid == 0) {
        *p.status = status;
        p.w.count[0] = status ? 0 : total;
    }
    if (status) return;
    if (p.op == OP_FREE) {
        for (uint32_t x = tid; alone && x < p.n * p.c.max_pages; x += PLAN_THREADS) free_place(p, x / p.c.max_pages, x % p.c.max_pages, err);
        return;
    }
    __syncthreads();
    for (uint32_t j = tid; j < total; j += PLAN_THREADS) {
        const uint32_t i = entry_of(p.w.first, p.n, j), k = j - p.w.first[i], page = p.w.page[j];
        const uint32_t s = static_cast<uint32_t>(changed[i]);
        uint32_t place = k;
        if (p.op == OP_GROW) place += pages_of(p.c, p.c.lens[s]);
        if (p.op == OP_FORK) place = static_cast<uint32_t>(p.num[i]) >> p.c.pshift;
        p.c.table[static_cast<size_t>(s) * p.c.max_pages + place] = static_cast<int32_t>(page);
        p.c.refs[page] = 1;
        if (p.op != OP_GROW) {
            const int32_t from = p.src.table[static_cast<size_t>(p.a[i]) * p.src.max_pages + place];
            p.w.from[j] = static_cast<uint32_t>(from);
            p.w.to[j] = page;
        }
    }
    if (p.op == OP_GROW) {
        __syncthreads();  // lens is read above
        for (uint32_t i = tid; i < p.n; i += PLAN_THREADS) p.c.lens[p.a[i]] += p.num[i];
    }
}

// The pages listed in from and to, every layer, COPY_CHUNK bytes a block
// and step.
__device__ void copy_pages(const Cache4& c, const Cache4& src, const PlanWork& w, uint32_t* err) {
    const uint32_t chunks = static_cast<uint32_t>((c.page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
    const uint64_t all = static_cast<uint64_t>(w.count[0]) * c.n_layers * chunks;
    for (uint64_t x = blockIdx.x; x < all; x += gridDim.x) {
        const uint32_t chunk = static_cast<uint32_t>(x % chunks), layer = static_cast<uint32_t>(x / chunks % c.n_layers);
        const uint64_t j = x / chunks / c.n_layers;
        const uint32_t from = w.from[j], to = w.to[j];
        if (from >= src.n_pages || to >= c.n_pages) {
            if (threadIdx.x == 0) atomicOr(err, PKB_DEVERR_ARGS);
            continue;
        }
        const size_t at = static_cast<size_t>(chunk) * COPY_CHUNK;
        const uint32_t words = static_cast<uint32_t>((c.page_bytes - at < COPY_CHUNK ? c.page_bytes - at : COPY_CHUNK) / 16);
        const uint4* x4 = reinterpret_cast<const uint4*>(src.pages + layer * src.layer_bytes + from * src.page_bytes + at);
        uint4* y4 = reinterpret_cast<uint4*>(c.pages + layer * c.layer_bytes + to * c.page_bytes + at);
        uint4 v[COPY_CHUNK / 16 / 256];
#pragma unroll
        for (int q = 0; q < static_cast<int>(COPY_CHUNK / 16 / 256); q++)
            if (threadIdx.x + q * 256 < words) v[q] = x4[threadIdx.x + q * 256];
#pragma unroll
        for (int q = 0; q < static_cast<int>(COPY_CHUNK / 16 / 256); q++)
            if (threadIdx.x + q * 256 < words) y4[threadIdx.x + q * 256] = v[q];
    }
}

// fork's and copy's bytes, and fork's shared pages; free's references.
__global__ void __launch_bounds__(256) apply_kernel(PlanArgs p, uint32_t* err) {
    pdl_trigger();
    pdl_wait();
    if (*p.status) return;
    for (uint32_t i = blockIdx.x; i < p.n; i += gridDim.x) {
        if (p.op == OP_FREE) {
            for (uint32_t j = threadIdx.x; j < p.c.max_pages; j += 256) free_place(p, i, j, err);
            continue;
        }
        if (p.op == OP_FORK) {
            const size_t from = static_cast<size_t>(p.a[i]) * p.c.max_pages, to = static_cast<size_t>(p.b[i]) * p.c.max_pages;
            const uint32_t whole = static_cast<uint32_t>(p.num[i]) >> p.c.pshift;
            for (uint32_t j = threadIdx.x; j < whole; j += 256) {
                const int32_t page = p.c.table[from + j];
                p.c.table[to + j] = page;
                if (page >= 0 && static_cast<uint32_t>(page) < p.c.n_pages) atomicAdd(p.c.refs + page, 1);
                else atomicOr(err, PKB_DEVERR_ARGS);
            }
        }
        if (threadIdx.x == 0) p.c.lens[p.b[i]] = p.num[i];
    }
    if (p.op != OP_FREE) copy_pages(p.c, p.src, p.w, err);
}

// compact: the holes below the count of used pages and the used pages from
// there on, each in order; the i-th of these goes to the i-th of those.
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(Cache4 c, PlanWork w, int32_t* used, int32_t* status) {
    __shared__ uint32_t buf[32];
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x;
    uint32_t count = 0;
    for (uint32_t p0 = tid * PLAN_REFS; p0 < c.n_pages; p0 += PLAN_THREADS * PLAN_REFS) {
        int32_t r[PLAN_REFS];
        load_refs(c, p0, r);
#pragma unroll
        for (int q = 0; q < PLAN_REFS; q++) count += p0 + q < c.n_pages && r[q] != 0;
    }
    uint32_t total;
    block_scan(count, &total, buf);
    uint32_t holes = 0, moves = 0;
    for (uint32_t q0 = 0; q0 < c.n_pages; q0 += PLAN_THREADS * PLAN_REFS) {
        const uint32_t p0 = q0 + tid * PLAN_REFS;
        int32_t r[PLAN_REFS];
        load_refs(c, p0, r);
        uint32_t h = 0, m = 0;
#pragma unroll
        for (int q = 0; q < PLAN_REFS; q++) {
            h += p0 + q < total && r[q] == 0;
            m += p0 + q >= total && p0 + q < c.n_pages && r[q] != 0;
        }
        uint32_t hs, ms;
        uint32_t hat = holes + block_scan(h, &hs, buf), mat = moves + block_scan(m, &ms, buf);
#pragma unroll
        for (int q = 0; q < PLAN_REFS; q++) {
            if (p0 + q < total && r[q] == 0) w.to[hat++] = p0 + q;
            if (p0 + q >= total && p0 + q < c.n_pages && r[q] != 0) w.from[mat++] = p0 + q;
        }
        holes += hs;
        moves += ms;
    }
    __syncthreads();
    for (uint32_t j = tid; j < moves; j += PLAN_THREADS) w.page[w.from[j]] = w.to[j];
    if (tid == 0) {
        w.count[0] = moves;
        w.count[1] = total;
        if (used) *used = static_cast<int32_t>(total);
        *status = PKB_CACHE4_DONE;
    }
}

__global__ void __launch_bounds__(256) compact_apply_kernel(Cache4 c, PlanWork w, uint32_t* err) {
    pdl_trigger();
    pdl_wait();
    const uint32_t moves = w.count[0], total = w.count[1];
    if (!moves) return;
    const size_t entries = static_cast<size_t>(c.max_seqs) * c.max_pages, first = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    for (size_t i = first; i < entries; i += static_cast<size_t>(gridDim.x) * 256) {
        const int32_t page = c.table[i];
        // a page from `total` on that a table names is in use, so it has a place
        if (page >= static_cast<int32_t>(total) && static_cast<uint32_t>(page) < c.n_pages) c.table[i] = static_cast<int32_t>(w.page[page]);
    }
    for (size_t j = first; j < moves; j += static_cast<size_t>(gridDim.x) * 256) {
        c.refs[w.to[j]] = c.refs[w.from[j]];
        c.refs[w.from[j]] = 0;
    }
    copy_pages(c, c, w, err);
}

__global__ void __launch_bounds__(256) reset_kernel(Cache4 c) {
    pdl_trigger();
    pdl_wait();
    const size_t first = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<size_t>(gridDim.x) * 256;
    for (size_t i = first; i < static_cast<size_t>(c.max_seqs) * c.max_pages; i += step) c.table[i] = -1;
    for (size_t i = first; i < c.max_seqs; i += step) c.lens[i] = 0;
    for (size_t i = first; i < c.n_pages; i += step) c.refs[i] = 0;
}

// ------------------------------------------------------------------- host --

size_t up256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

size_t plan_layout(const pkb_cache4* c, uint8_t* base, PlanWork* w) {
    size_t at = 0;
    auto take = [&](size_t n) {
        uint32_t* p = reinterpret_cast<uint32_t*>(base + at);
        at += up256(n * 4);
        return p;
    };
    w->count = take(64);
    w->mark = take(c->max_seqs);
    w->first = take(static_cast<size_t>(c->max_seqs) + 1);
    w->page = take(c->n_pages);
    w->from = take(c->n_pages);
    w->to = take(c->n_pages);
    return at;
}

bool is_aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int cuda_error(cudaError_t e, const char* who) {
    return set_error(e == cudaErrorMemoryAllocation ? PKB_ENOMEM : PKB_ECUDA, "%s launch: %s", who, cudaGetErrorString(e));
}

int check_plan(const pkb_cache4* c, const char* who, int32_t* status, void* work, size_t work_bytes, Cache4* v, PlanWork* w) {
    int rc = c4_view(c, who, v);
    if (rc) return rc;
    if (!status || !work) return set_error(PKB_EINVAL, "%s: null pointer", who);
    if (!is_aligned(status, 4) || !is_aligned(work, 256)) return set_error(PKB_EINVAL, "%s: misaligned status or work area", who);
    const size_t need = plan_layout(c, static_cast<uint8_t*>(work), w);
    if (work_bytes < need) return set_error(PKB_EINVAL, "%s: work area of %zu bytes, %zu needed", who, work_bytes, need);
    return PKB_OK;
}

int page_op(cudaStream_t stream, int op, const char* who, const pkb_cache4* c, const pkb_cache4* src, const int32_t* a,
            const int32_t* b, const int32_t* num, uint32_t n, int32_t* status, void* work, size_t work_bytes) {
    PlanArgs p = {};
    int rc = check_plan(c, who, status, work, work_bytes, &p.c, &p.w);
    if (rc) return rc;
    p.src = p.c;
    if (src != c) {
        if ((rc = c4_view(src, who, &p.src))) return rc;
        if (src->n_layers != c->n_layers || src->page_tokens != c->page_tokens || src->n_heads != c->n_heads ||
            src->head_dim != c->head_dim)
            return set_error(PKB_EINVAL, "%s: the two caches differ in layers, page_tokens, heads or head_dim", who);
    }
    if (n > c->max_seqs) return set_error(PKB_EINVAL, "%s: %u entries for %u sequences", who, n, c->max_seqs);
    const bool two = op == OP_FORK || op == OP_COPY;
    if (n && (!a || (two && !b) || (op != OP_FREE && !num))) return set_error(PKB_EINVAL, "%s: null pointer", who);
    if (!is_aligned(a, 4) || !is_aligned(b, 4) || !is_aligned(num, 4)) return set_error(PKB_EINVAL, "%s: misaligned list", who);
    int sms;
    uint32_t* err;
    if ((rc = current_device_info(&sms, &err))) return rc;
    p.a = a;
    p.b = b;
    p.num = num;
    p.n = n;
    p.op = op;
    p.status = status;
    // a few rows' pages are freed by the block that checked them: a second launch takes as long as some 16,000 places
    const bool alone = op == OP_FREE && static_cast<uint64_t>(n) * c->max_pages <= 16384;
    cudaError_t e = c4_launch(plan_kernel, 1, PLAN_THREADS, 0, stream, p, alone, err);
    if (e != cudaSuccess) return cuda_error(e, who);
    count_launch();
    if (op == OP_GROW || alone || !n) return PKB_OK;
    // a block an entry, or enough blocks that a copy keeps every SM's loads in flight
    const uint64_t most = op == OP_FREE ? n : n + static_cast<uint64_t>(op == OP_FORK ? n : c->n_pages) * c->n_layers *
                                                      ((p.c.page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
    const uint32_t grid = static_cast<uint32_t>(most < 8u * sms ? most : 8u * sms);
    e = c4_launch(apply_kernel, grid, 256, 0, stream, p, err);
    if (e != cudaSuccess) return cuda_error(e, who);
    count_launch();
    return PKB_OK;
}

template <typename T, int NB>
cudaError_t launch_rows(bool append, bool vec, void* k, void* v, const RowArgs& a, cudaStream_t s) {
    const size_t warps = 2 * static_cast<size_t>(a.slots) * a.c.heads;
    const dim3 grid(static_cast<uint32_t>((warps + ROW_WARPS - 1) / ROW_WARPS)), block(ROW_WARPS * 32);
    const T *kc = static_cast<const T*>(k), *vc = static_cast<const T*>(v);
    T *ko = static_cast<T*>(k), *vo = static_cast<T*>(v);
    if (append)
        return vec ? c4_launch(append_kernel<T, NB, true>, grid, block, 0, s, kc, vc, a)
                   : c4_launch(append_kernel<T, NB, false>, grid, block, 0, s, kc, vc, a);
    return vec ? c4_launch(read_kernel<T, NB, true>, grid, block, 0, s, ko, vo, a)
               : c4_launch(read_kernel<T, NB, false>, grid, block, 0, s, ko, vo, a);
}

template <typename T>
cudaError_t launch_rows_dk(bool append, bool vec, void* k, void* v, const RowArgs& a, cudaStream_t s) {
    switch (a.c.dk) {
        case 32: return launch_rows<T, 1>(append, vec, k, v, a, s);
        case 64: return launch_rows<T, 2>(append, vec, k, v, a, s);
        case 96: return launch_rows<T, 3>(append, vec, k, v, a, s);
        case 128: return launch_rows<T, 4>(append, vec, k, v, a, s);
        default: return launch_rows<T, 8>(append, vec, k, v, a, s);
    }
}

int rows_call(cudaStream_t stream, bool append, const pkb_cache4* c, uint32_t layer, void* k, size_t ks, void* v, size_t vs,
              int type, const int32_t* seqs, const int32_t* starts, uint32_t n, uint32_t rows, const int32_t* status) {
    const char* who = append ? "cache4_append" : "cache4_read";
    RowArgs a = {};
    int rc = c4_view(c, who, &a.c);
    if (rc) return rc;
    if ((rc = c4_check_type(type, who))) return rc;
    if (layer >= c->n_layers) return set_error(PKB_EINVAL, "%s: layer %u of %u", who, layer, c->n_layers);
    if (!n || !rows) return PKB_OK;
    if (!k || !v || !seqs || !starts) return set_error(PKB_EINVAL, "%s: null pointer", who);
    const size_t width = static_cast<size_t>(c->n_heads) * c->head_dim, size = c4_type_bytes(type);
    if (rows > 1 && (ks < width || vs < width)) return set_error(PKB_EINVAL, "%s: a row stride below %zu values", who, width);
    if (rows == 1) ks = vs = width;
    if (!is_aligned(k, size) || !is_aligned(v, size) || !is_aligned(seqs, 4) || !is_aligned(starts, 4) || !is_aligned(status, 4))
        return set_error(PKB_EINVAL, "%s: misaligned buffer", who);
    const uint64_t slots = static_cast<uint64_t>(rows) / C4_UNIT + 2 * static_cast<uint64_t>(n);
    if (rows > INT_MAX || slots > UINT_MAX || slots * 2 * c->n_heads / ROW_WARPS >= INT_MAX)
        return set_error(PKB_EINVAL, "%s: %u rows of %u sequences are too many for one launch", who, rows, n);
    uint32_t* err;
    int sms;
    if ((rc = current_device_info(&sms, &err))) return rc;
    a.seqs = seqs;
    a.starts = starts;
    a.status = status;
    a.err = err;
    a.ks = ks;
    a.vs = vs;
    a.layer = layer;
    a.n = n;
    a.rows = rows;
    a.slots = static_cast<uint32_t>(slots);
    const bool vec = is_aligned(k, 16) && is_aligned(v, 16) && ks * size % 16 == 0 && vs * size % 16 == 0;
    const cudaError_t e = type == PKB_F32   ? launch_rows_dk<float>(append, vec, k, v, a, stream)
                          : type == PKB_F16 ? launch_rows_dk<__half>(append, vec, k, v, a, stream)
                                            : launch_rows_dk<__nv_bfloat16>(append, vec, k, v, a, stream);
    if (e != cudaSuccess) return cuda_error(e, who);
    count_launch();
    return PKB_OK;
}

}  // namespace

int c4_check_type(int type, const char* who) {
    if (type != PKB_F32 && type != PKB_F16 && type != PKB_BF16) return set_error(PKB_EINVAL, "%s: type %d", who, type);
    return PKB_OK;
}

int c4_view(const pkb_cache4* c, const char* who, Cache4* v) {
    if (!c) return set_error(PKB_EINVAL, "%s: null cache", who);
    const size_t page = pkb_cache4_page_bytes(c->page_tokens, c->n_heads, c->head_dim);
    if (!page)
        return set_error(PKB_EINVAL, "%s: pages of %u tokens, %u heads of %u: 16 to 256 tokens, a power of two; heads of 32, 64, 96, 128 or 256",
                         who, c->page_tokens, c->n_heads, c->head_dim);
    if (!c->n_layers || !c->n_pages || !c->max_seqs || !c->max_pages || c->n_pages > INT_MAX || c->max_seqs > INT_MAX ||
        static_cast<uint64_t>(c->max_pages) * c->page_tokens > 1u << 30)
        return set_error(PKB_EINVAL, "%s: %u layers, %u pages, %u sequences of up to %u pages", who, c->n_layers, c->n_pages,
                         c->max_seqs, c->max_pages);
    if (!c->pages || !c->table || !c->lens || !c->refs) return set_error(PKB_EINVAL, "%s: null pointer in the cache", who);
    if (!is_aligned(c->pages, 16) || !is_aligned(c->table, 4) || !is_aligned(c->lens, 4) || !is_aligned(c->refs, 4))
        return set_error(PKB_EINVAL, "%s: the cache's pages must be 16-byte aligned, its lists 4-byte", who);
    v->pages = c->pages;
    v->table = c->table;
    v->lens = c->lens;
    v->refs = c->refs;
    v->n_layers = c->n_layers;
    v->n_pages = c->n_pages;
    v->max_seqs = c->max_seqs;
    v->max_pages = c->max_pages;
    v->heads = c->n_heads;
    v->dk = c->head_dim;
    v->pshift = 4;
    while (1u << v->pshift < c->page_tokens) v->pshift++;
    v->unit_bytes = 18 * c->head_dim;
    v->head_bytes = static_cast<size_t>(c->page_tokens / C4_UNIT) * v->unit_bytes;
    v->page_bytes = page;
    v->layer_bytes = page * c->n_pages;
    return PKB_OK;
}

}  // namespace pkb

using namespace pkb;

extern "C" {

size_t pkb_cache4_page_bytes(uint32_t page_tokens, uint32_t n_heads, uint32_t head_dim) {
    if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1))) return 0;
    if (head_dim != 32 && head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 256) return 0;
    if (!n_heads || n_heads > 65535) return 0;
    return static_cast<size_t>(page_tokens / 16) * 18 * head_dim * n_heads;
}

size_t pkb_cache4_work_bytes(const pkb_cache4* c) {
    PlanWork w;
    if (!c || !c->n_pages || !c->max_seqs) return 0;
    return plan_layout(c, nullptr, &w);
}

int pkb_cache4_reset_dev(void* stream, const pkb_cache4* c) {
    Cache4 v;
    int rc = c4_view(c, "cache4_reset", &v), sms;
    uint32_t* err;
    if (rc || (rc = current_device_info(&sms, &err))) return rc;
    const cudaError_t e = c4_launch(reset_kernel, static_cast<uint32_t>(2 * sms), 256, 0, static_cast<cudaStream_t>(stream), v);
    if (e != cudaSuccess) return cuda_error(e, "cache4_reset");
    count_launch();
    return PKB_OK;
}

int pkb_cache4_grow_dev(void* stream, const pkb_cache4* c, const int32_t* seqs, const int32_t* add, uint32_t n,
                        int32_t* status, void* work, size_t work_bytes) {
    return page_op(static_cast<cudaStream_t>(stream), OP_GROW, "cache4_grow", c, c, seqs, nullptr, add, n, status, work, work_bytes);
}

int pkb_cache4_fork_dev(void* stream, const pkb_cache4* c, const int32_t* src, const int32_t* dst, const int32_t* len,
                        uint32_t n, int32_t* status, void* work, size_t work_bytes) {
    return page_op(static_cast<cudaStream_t>(stream), OP_FORK, "cache4_fork", c, c, src, dst, len, n, status, work, work_bytes);
}

int pkb_cache4_copy_dev(void* stream, const pkb_cache4* to, const pkb_cache4* from, const int32_t* src,
                        const int32_t* dst, const int32_t* len, uint32_t n, int32_t* status, void* work,
                        size_t work_bytes) {
    return page_op(static_cast<cudaStream_t>(stream), OP_COPY, "cache4_copy", to, from, src, dst, len, n, status, work, work_bytes);
}

int pkb_cache4_free_dev(void* stream, const pkb_cache4* c, const int32_t* seqs, uint32_t n, int32_t* status,
                        void* work, size_t work_bytes) {
    return page_op(static_cast<cudaStream_t>(stream), OP_FREE, "cache4_free", c, c, seqs, nullptr, nullptr, n, status, work, work_bytes);
}

int pkb_cache4_compact_dev(void* stream, const pkb_cache4* c, int32_t* used, int32_t* status, void* work,
                           size_t work_bytes) {
    const char* who = "cache4_compact";
    Cache4 v;
    PlanWork w;
    int rc = check_plan(c, who, status, work, work_bytes, &v, &w), sms;
    if (rc) return rc;
    if (!is_aligned(used, 4)) return set_error(PKB_EINVAL, "%s: misaligned list", who);
    uint32_t* err;
    if ((rc = current_device_info(&sms, &err))) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = c4_launch(compact_plan_kernel, 1, PLAN_THREADS, 0, s, v, w, used, status);
    if (e != cudaSuccess) return cuda_error(e, who);
    count_launch();
    e = c4_launch(compact_apply_kernel, static_cast<uint32_t>(8 * sms), 256, 0, s, v, w, err);
    if (e != cudaSuccess) return cuda_error(e, who);
    count_launch();
    return PKB_OK;
}

int pkb_cache4_append_dev(void* stream, const pkb_cache4* c, uint32_t layer, const void* k, size_t ks, const void* v,
                          size_t vs, int type, const int32_t* seqs, const int32_t* starts, uint32_t n, uint32_t rows) {
    return rows_call(static_cast<cudaStream_t>(stream), true, c, layer, const_cast<void*>(k), ks, const_cast<void*>(v), vs,
                     type, seqs, starts, n, rows, nullptr);
}

int pkb_cache4_append_if_dev(void* stream, const pkb_cache4* c, uint32_t layer, const void* k, size_t ks, const void* v,
                             size_t vs, int type, const int32_t* seqs, const int32_t* starts, uint32_t n, uint32_t rows,
                             const int32_t* status) {
    return rows_call(static_cast<cudaStream_t>(stream), true, c, layer, const_cast<void*>(k), ks, const_cast<void*>(v), vs,
                     type, seqs, starts, n, rows, status);
}

int pkb_cache4_read_dev(void* stream, const pkb_cache4* c, uint32_t layer, void* k, size_t ks, void* v, size_t vs,
                        int type, const int32_t* seqs, const int32_t* starts, uint32_t n, uint32_t rows) {
    return rows_call(static_cast<cudaStream_t>(stream), false, c, layer, k, ks, v, vs, type, seqs, starts, n, rows, nullptr);
}

}  // extern "C"
