// Attention over a cache held in 4 bits, few rows over long sequences
// (include/pktito_b200.h, pkb_attention_cache4_dev).
//
// The mathematics. For a sequence and a cached head, the rows (query heads
// that share it, times the call's tokens) are columns of products whose
// other operand is the cache:
//     S^T [keys x rows] = K Q^T,  P = 2^(scale log2e S - m),
//     O^T [dk x rows]  += V^T P,  l += sum P,
// one pass over the keys with the running maximum m and sum l. K and V are
// the 16-row operand of mma.m16n8k16, so eight rows fill an instruction and
// a step of decoding with up to eight query heads a cached head wastes
// none. The codes become exact bf16 values in registers, three instructions
// a pair (pkb_cache4.cuh); their order in the cache is that operand's, so
// no value crosses a lane. V is exact, and P is two bf16 parts for f16 and
// bf16 rows (16 bits), three for float rows (24). One part, P rounded to bf16
// before it meets V, is as far off as o's own rounding: 2.3e-3 of the result for
// bf16 rows against 1.65e-3 for two parts and for weights in float, of which
// 1.65e-3 is o's; it takes a tenth less time (64 sequences 49.9 us against 55).
//
// The split. A team of up to 16 cached heads' warps goes over the same
// tiles of 32 keys side by side, each for its own head, so that what they
// fetch lies together in a page. All (sequence, team, block of rows) items'
// tiles are laid end to end and divided evenly over all teams of warps on the
// GPU, whatever the sequences' lengths: a share begins and ends inside
// items. Each warp fetches for itself (bulk copies of whole units, 18 dk
// bytes, into a ring of its own, some tiles ahead), so warps never wait for
// one another. An item that one share has whole is written at once; of
// the others each share leaves its part (m, l, O) in the work area, and a
// second kernel joins an item's parts in a fixed order.
//
// What bounds it. Neither the cache's bytes (1.125 dk a token and cached head) nor
// the issue slots (57 % of them), but each warp's chain from the codes to the
// products: a tile of 32 keys of a head of 128 is some 560 instructions of a warp,
// seven cycles each, of which two are fixed latencies and one a busy pipe, and the
// four warps that a quarter of an SM has registers for do not cover that.
// One step of 64 sequences of up to 4,099 tokens (161 MB, 8 heads of 128 with 4
// query heads each, bf16): 55 us with its join, 2.9 TB/s; three sequences of up
// to 120,001 tokens with 8 query heads each: 62 us, 3.2 TB/s. Of that some 7 us pass
// before the first tile (the entries' lengths, their scan, the first pages) and
// 5 in the join: short calls (12 us for one sequence of 377 tokens) are nothing else.
// (With weights in one part, 52 us then: scaled bf16 values for K too 66 us for
// the 64 sequences, one warp that fetches for all of a block's 55.)

#include <atomic>
#include <climits>
#include <mutex>
#include <type_traits>

#include "pkb_attn4.cuh"
#include "pkb_internal.h"

namespace pkb {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int JOIN_WARPS = 8;
constexpr int TILE = 32;            // keys of a tile: two units
constexpr uint32_t MAX_ENTRIES = 1024;  // sequences of one launch
constexpr uint32_t MAX_TEAM = 16;       // (teams of 4 and 8 take as long: 64 sequences of 2,048 tokens, 16 heads, 88 us)
constexpr uint32_t SPLIT_ROWS = 1024;   // rows of an entry and cached head that may be split along the keys
constexpr int MAX_GRID = 160;
constexpr int MAX_WORKERS = 16;

// Warps of a block, one block an SM. Sixteen leave a thread 128 registers,
// eight 255.
template <int NB, int NT> __host__ __device__ constexpr int workers() { return NB * NT <= 4 ? 16 : 8; }
template <int NB, int NT> __host__ __device__ constexpr int stages() { return NB <= 2 ? 4 : NB * NT == 4 || NB == 8 ? 2 : 3; }
template <int NB> __host__ __device__ constexpr int tile_bytes() { return 2 * 18 * 32 * NB; }
template <int NB, int NT> __host__ __device__ constexpr int part_regs() { return NT * (NB * 8 + 4); }  // a lane's of one part

// `total` places over `n` shares, the first ones one more than the others.
struct Split {
    uint32_t n, each, more;
    __device__ __forceinline__ Split(uint32_t total, uint32_t most) {
        n = total < most ? total : most;
        each = n ? total / n : 0;
        more = n ? total - each * n : 0;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t s) const { return s * each + (s < more ? s : more); }
    __device__ __forceinline__ uint32_t of(uint32_t x) const {
        const uint32_t wide = more * (each + 1);
        return x < wide ? x / (each + 1) : more + (x - wide) / each;
    }
};

// A lane's columns are rows 8 j + 2 t + {0, 1} of a block of 8 NT: their
// token in the entry, and what they may see. All of it is cheap to make
// again, so none of it is held over the loop on the tiles.
struct Column {
    uint32_t r, tok;
    bool valid;
    int32_t lo, hi;  // keys [lo, hi)
};

template <int NT>
__device__ __forceinline__ Column column(const Attn4Args& a, const Entry& e, uint32_t block, int i) {
    Column c;
    c.r = block * (8 * NT) + i / 2 * 8 + 2 * (threadIdx.x & 3) + i % 2;
    c.tok = c.r / a.G;
    c.valid = c.tok < e.rows;
    const Keys k = keys_of(a, e, c.tok);
    c.lo = k.lo;
    c.hi = c.valid ? k.hi : 0;
    return c;
}

template <typename T, int NB, int NT>
__device__ __forceinline__ void write_rows(const Attn4Args& a, const Entry& e, uint32_t h, uint32_t block,
                                           const float (&o)[2 * NB][NT][4], const float (&l)[2 * NT]) {
    const uint32_t g = (threadIdx.x & 31) / 4;
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
        const Column c = column<NT>(a, e, block, i);
        if (!c.valid) continue;
        T* out = static_cast<T*>(a.o) + static_cast<size_t>(e.r0 + c.tok) * a.os + (h * a.G + c.r - c.tok * a.G) * (NB * 32) + g;
        // V came as quarters; a row that sees nothing has sum 0 and is zeros; a NaN sum gives NaNs
        const float inv = l[i] == 0.0f ? 0.0f : __fdiv_rn(4.0f, l[i]);
#pragma unroll
        for (int m = 0; m < 2 * NB; m++)
#pragma unroll
            for (int r = 0; r < 2; r++) out[m * 16 + r * 8] = c4_round<T>(__fmul_rn(o[m][i / 2][i % 2 + 2 * r], inv));
    }
}

// Sums over the eight lanes that hold a column's keys.
__device__ __forceinline__ float column_sum(float x) {
    x += __shfl_xor_sync(FULL, x, 4);
    x += __shfl_xor_sync(FULL, x, 8);
    x += __shfl_xor_sync(FULL, x, 16);
    return x;
}
__device__ __forceinline__ float column_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(FULL, x, 4));
    x = fmaxf(x, __shfl_xor_sync(FULL, x, 8));
    x = fmaxf(x, __shfl_xor_sync(FULL, x, 16));
    return x;
}

// NB words (or scale halves, as words) from shared memory, as wide as they lie
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
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

// A block's rows of q as the second operand of the products with K, which
// are taken in f16: K's codes are whole numbers there (c4_whole), fewer
// instructions than scaled bf16 values, and their scales multiply the sums of
// a block of 32. (Codes + 8, and + 72 in every other pair, with sums that start
// at what that adds, save four of a word's instructions and cost as many moves:
// 16 rows a head 48.0 us against 46.2, single tokens the same. And the large sums cut
// off what small values of q add.) A row is brought to a largest value in [2^14, 2^15)
// by a power of two. What that and the softmax's scale are together, up to 2^0,
// goes into K's scales before they multiply the sums, which alone pass a float's
// range for K from 2^104 on; the rest multiplies the scores (23 float rows of
// 32 sequences 26.7 -> 27.7 us in a graph, single tokens 1 %). A row is one f16 (bf16 and f16
// rows) or two (float rows, PARTS 3): exact but for 2^-24 of a float, and for
// 2^-39 of the row's largest value.
template <int NB, int NT, int PARTS>
struct Query {
    static constexpr int P = PARTS == 3 ? 2 : 1;
    uint32_t w[NB][2][NT][P][2];
    uint64_t k_scale[NT], scale[NT];  // of each pair of the lane's columns
};

template <typename T, int NB, int NT, int PARTS>
__device__ __forceinline__ void load_query(const Attn4Args& a, const Entry& e, uint32_t h, uint32_t block, Query<NB, NT, PARTS>& q) {
    constexpr int P = Query<NB, NT, PARTS>::P;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const uint32_t r = block * (8 * NT) + j * 8 + g, tok = r / a.G;
        const T* qp = static_cast<const T*>(a.q) + static_cast<size_t>(e.r0 + tok) * a.qs + (h * a.G + r - tok * a.G) * (NB * 32) + 8 * t;
        float f[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int y = 0; y < 8; y++) f[b][y] = 0.0f;
            if (tok < e.rows) {
                if (a.vec) c4_load8<T, true>(qp + b * 32, f[b]);
                else c4_load8<T, false>(qp + b * 32, f[b]);
            }
        }
        float top = 0.0f;  // NaNs pass the maximum by and stay NaNs below
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int y = 0; y < 8; y++) top = fmaxf(top, fabsf(f[b][y]));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
        // 2^(14 - x) for a largest value in [2^x, 2^(x+1)); an infinite one makes the row NaNs
        const int x = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -110);
        const float up = __uint_as_float(x == 128 ? 0x7FC00000u : static_cast<uint32_t>(141 - x) << 23);
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int y = 0; y < 4; y++) {
                uint32_t parts[P];
                f16_parts<P>(f[b][2 * y] * up, f[b][2 * y + 1] * up, parts);
#pragma unroll
                for (int z = 0; z < P; z++) q.w[b][y / 2][j][z][y % 2] = parts[z];
            }
        }
        // scale 2^(x - 14) as a power of two in [2^-126, 1] and the rest
        const int e0 = min(x, 127) - 14, e1 = max(min(e0 + max(static_cast<int>(__float_as_uint(a.scale) >> 23 & 255), 1) - 127, 0), -126);
        const float k_scale = __uint_as_float(static_cast<uint32_t>(e1 + 127) << 23), rest = fminf(fmaxf(ldexpf(a.scale, e0 - e1), -3.0e38f), 3.0e38f);
        const int c0 = static_cast<int>(2 * t * 4), c1 = c0 + 4;
        q.k_scale[j] = pack2(__shfl_sync(FULL, k_scale, c0), __shfl_sync(FULL, k_scale, c1));
        q.scale[j] = pack2(__shfl_sync(FULL, rest, c0), __shfl_sync(FULL, rest, c1));
    }
}

// Scores of one unit: S^T[keys g, g + 8][columns 2t, 2t + 1].
template <int NB, int NT, int PARTS>
__device__ __forceinline__ void unit_scores(const uint8_t* unit, const Query<NB, NT, PARTS>& q, float (&s)[NT][4]) {
    constexpr int DK = NB * 32, P = Query<NB, NT, PARTS>::P;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    uint32_t w[2][NB];
    lds_words<NB>(unit + (g * 4 + t) * NB * 4, w[0]);
    lds_words<NB>(unit + ((g + 8) * 4 + t) * NB * 4, w[1]);
    uint32_t sc[2][(NB + 1) / 2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const uint8_t* at = unit + 16 * DK + (g + 8 * r) * NB * 2;
        if constexpr (NB % 2 == 0) {
            lds_words<NB / 2>(at, sc[r]);
        } else {
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                sc[r][b / 2] = *reinterpret_cast<const uint16_t*>(at + 2 * b);
                if (b + 1 < NB) sc[r][b / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + 2 * b + 2)) << 16;
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; b++) {
        uint64_t k[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const float x = __uint_as_float(b % 2 ? sc[r][b / 2] & 0xFFFF0000u : sc[r][b / 2] << 16);
            k[r] = pack2(x, x);
        }
        const uint32_t a0[4] = {c4_whole<0>(w[0][b]), c4_whole<0>(w[1][b]), c4_whole<1>(w[0][b]), c4_whole<1>(w[1][b])};
        const uint32_t a1[4] = {c4_whole<2>(w[0][b]), c4_whole<2>(w[1][b]), c4_whole<3>(w[0][b]), c4_whole<3>(w[1][b])};
#pragma unroll
        for (int j = 0; j < NT; j++) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = P - 1; p >= 0; p--) {
                mma_f16(d, a0, q.w[b][0][j][p][0], q.w[b][0][j][p][1]);
                mma_f16(d, a1, q.w[b][1][j][p][0], q.w[b][1][j][p][1]);
            }
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint64_t ks = mul2_r<0>(k[r], q.k_scale[j]), y = pack2(d[2 * r], d[2 * r + 1]);
                uint64_t sum = b ? fma2_r<0>(y, ks, pack2(s[j][2 * r], s[j][2 * r + 1])) : mul2_r<0>(y, ks);
                if (b + 1 == NB) sum = mul2_r<0>(sum, q.scale[j]);
                unpack2(sum, s[j][2 * r], s[j][2 * r + 1]);
            }
        }
    }
}

// One tile of two units at `buf`: its scores, the softmax's step, its values.
// mask: some key of it is hidden from some row, or lies past the last one
// that was fetched (limit).
template <int NB, int NT, int PARTS>
__device__ __forceinline__ void tile_step(bool mask, const Attn4Args& args, const Entry& e, uint32_t block, uint8_t* buf,
                                          const Query<NB, NT, PARTS>& q, int32_t key0, int32_t limit,
                                          float (&o)[2 * NB][NT][4], float (&m)[2 * NT], float (&l)[2 * NT]) {
    constexpr int DK = NB * 32;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    if (mask && key0 + TILE > limit) {
        // V's scales past the limit may be anything, and 0 times a NaN is one: they become zeros where they lie
        for (uint32_t x = lane; x < 2 * NB * C4_UNIT; x += 32) {
            const uint32_t u = x / (NB * C4_UNIT), at = x % (NB * C4_UNIT);
            if (key0 + static_cast<int32_t>(C4_UNIT * u + at % C4_UNIT) >= limit)
                *reinterpret_cast<uint16_t*>(buf + u * 18 * DK + 17 * DK + 2 * at) = 0;
        }
        fence_async_smem();  // before a later copy into this place
        __syncwarp();
    }
    float s[2][NT][4];
    unit_scores<NB, NT, PARTS>(buf, q, s[0]);
    unit_scores<NB, NT, PARTS>(buf + 18 * DK, q, s[1]);
    bool above = false;
    if (mask) {
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) {
            const Column c = column<NT>(args, e, block, i);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int32_t key = key0 + 16 * u + static_cast<int32_t>(g) + 8 * r;
                    if (key < c.lo || key >= c.hi) s[u][i / 2][i % 2 + 2 * r] = NEG_INF;
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
        const float limit = m[i] + 8.0f;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 2; r++) above |= s[u][i / 2][i % 2 + 2 * r] > limit;
    }
    // The maximum is raised only where some score passes it by 8: sums and
    // weights then stay below 2^8 times the keys, far inside a float, and
    // most tiles need one vote instead of the reductions.
    if (__any_sync(FULL, above)) {
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) {
            float top = m[i];
#pragma unroll
            for (int u = 0; u < 2; u++) top = fmaxf(top, fmaxf(s[u][i / 2][i % 2], s[u][i / 2][i % 2 + 2]));
            top = column_max(top);
            const float f = rescale(m[i], top);
            m[i] = top;
            l[i] *= f;
#pragma unroll
            for (int d = 0; d < 2 * NB; d++) {
                o[d][i / 2][i % 2] *= f;
                o[d][i / 2][i % 2 + 2] *= f;
            }
        }
    }
    uint32_t p[2][NT][2][PARTS];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float m0 = m[2 * j] == NEG_INF ? 0.0f : m[2 * j], m1 = m[2 * j + 1] == NEG_INF ? 0.0f : m[2 * j + 1];
                const float p0 = exp2_fast(__fsub_rn(s[u][j][2 * r], m0)), p1 = exp2_fast(__fsub_rn(s[u][j][2 * r + 1], m1));
                l[2 * j] += p0;
                l[2 * j + 1] += p1;
                bf16_parts<PARTS>(p0, p1, p[u][j][r]);
#pragma unroll
                for (int x = 0; x < PARTS; x++) p[u][j][r][x] = transpose8(p[u][j][r][x]);
            }
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float fresh[2][NT][4];
        if constexpr (PARTS == 3) {
#pragma unroll
            for (int d = 0; d < 2; d++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) fresh[d][j][x] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint8_t* unit = buf + u * 18 * DK;
            const uint2 w = *reinterpret_cast<const uint2*>(unit + 8 * DK + ((b * 8 + g) * 4 + t) * 8);
            uint32_t s2[2], ms[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                s2[c] = *reinterpret_cast<const uint32_t*>(unit + 17 * DK + (b * C4_UNIT + 8 * c + 2 * t) * 2);
                ms[c] = c4_m6(s2[c]);
            }
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const uint32_t x = d ? w.y : w.x;
                uint32_t a[4];
                a[0] = c4_quarter<0>(x, s2[0], ms[0]);
                a[1] = c4_quarter<1>(x, s2[0], ms[0]);
                a[2] = c4_quarter<2>(x, s2[1], ms[1]);
                a[3] = c4_quarter<3>(x, s2[1], ms[1]);
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int y = PARTS - 1; y >= 0; y--)
                        mma_bf16(PARTS == 3 ? fresh[d][j] : o[2 * b + d][j], a, p[u][j][0][y], p[u][j][1][y]);
            }
        }
        if constexpr (PARTS == 3) {
#pragma unroll
            for (int d = 0; d < 2; d++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) o[2 * b + d][j][x] = __fadd_rn(o[2 * b + d][j][x], fresh[d][j][x]);
        }
    }
}

template <typename T, int NB, int NT, int PARTS>
__global__ void __launch_bounds__(workers<NB, NT>() * 32, 1) split_kernel(Attn4Args a) {
    constexpr int DK = NB * 32, WORKERS = workers<NB, NT>(), THREADS = WORKERS * 32, STAGES = stages<NB, NT>(), BYTES = tile_bytes<NB>();
    constexpr int EACH = (MAX_ENTRIES + THREADS - 1) / THREADS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[WORKERS][STAGES];
    __shared__ uint64_t sums[WORKERS];
    __shared__ uint32_t most[WORKERS];
    __shared__ volatile int gave_up;
    Entry* entries = reinterpret_cast<Entry*>(smem + WORKERS * STAGES * BYTES);
    uint32_t* base = reinterpret_cast<uint32_t*>(entries + a.n);  // each entry's first place, or item where shares take whole ones
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (lane == 0) {
        for (int i = 0; i < STAGES; i++) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
    }
    if (tid == 0) gave_up = 0;
    pdl_trigger();
    pdl_wait();
    // places and items (in the upper half) before each entry, and the longest item's places
    uint64_t before[EACH], own = 0;
    uint32_t longest = 0;
#pragma unroll
    for (int x = 0; x < EACH; x++) {
        const uint32_t i = tid * EACH + x;
        before[x] = own;
        if (i < a.n) {
            const Entry e = load_entry(a, i);
            entries[i] = e;
            const uint64_t items = e.places ? a.teams * e.blocks<NT>(a) : 0;
            own += items * e.places + (items << 32);
            longest = max(longest, e.places);
        }
    }
    uint64_t scan = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint64_t y = __shfl_up_sync(FULL, scan, d);
        if (lane >= static_cast<uint32_t>(d)) scan += y;
    }
    longest = __reduce_max_sync(FULL, longest);
    if (lane == 31) sums[warp] = scan, most[warp] = longest;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < WORKERS; w++) {
        if (w == warp) scan += total - own;
        total += sums[w];
        longest = max(longest, most[w]);
    }
    // Where no item is longer than one and a half shares, shares take whole
    // items: there is nothing to join then (200 sequences of 512 tokens, 8
    // heads of 64, 4 bf16 rows each: 30.9 us in equal shares, 29.8 in whole items;
    // 40 of 700 tokens, heads of 128, one row each: 20.4 and 35.8).
    const uint32_t room = min(gridDim.x * WORKERS / a.team, a.max_shares), places = static_cast<uint32_t>(total);
    const bool whole = 2ull * longest * room <= 3ull * places;
#pragma unroll
    for (int x = 0; x < EACH; x++) {
        const uint32_t i = tid * EACH + x;
        if (i < a.n) base[i] = static_cast<uint32_t>(whole ? (scan + before[x]) >> 32 : scan + before[x]);
    }
    if (tid == 0) base[a.n] = whole ? static_cast<uint32_t>(total >> 32) : places;
    __syncthreads();
    const Split split(whole ? static_cast<uint32_t>(total >> 32) : places, room);
    // where a place lies: its entry, its item of that, and its place in the item
    struct Item {
        uint32_t entry, head0, block, place, places;
        uint32_t stop, next;  // the share's last place of it and one, and where its next item begins
    };
    auto item_at = [&](uint32_t x, uint32_t end) {
        Item it;
        uint32_t lo = 0, hi = a.n;  // thirty-two probes a step
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
            const uint32_t last = 31 - __clz(__ballot_sync(FULL, i < hi && base[i] <= x) | 1u);
            lo += last * step;
            hi = min(lo + step, hi);
        }
        it.entry = lo;
        const Entry& e = entries[lo];
        it.places = e.places;
        it.place = x - base[lo];
        it.block = it.head0 = 0;
        const uint32_t each = whole ? 1 : it.places;
        if (it.place >= each) {
            const uint32_t i = it.place / each, blocks = e.blocks<NT>(a), t = i / blocks;
            it.place -= i * each;
            it.block = i - t * blocks;
            it.head0 = t * a.team;
        }
        it.stop = whole ? it.places : min(it.places, it.place + (end - x));
        it.next = x + (whole ? 1 : it.stop - it.place);
        return it;
    };

    // a team's warps lie on neighbouring SMs, and so do shares
    const uint32_t v = warp * gridDim.x + blockIdx.x, share = v / a.team, member = v - share * a.team;
    uint8_t* ring = smem + warp * STAGES * BYTES;
    if (share < split.n) {
        uint32_t x = split.begin(share);
        const uint32_t end = split.begin(share + 1);
        // What is fetched next, STAGES tiles ahead of what is computed: lanes
        // 0 and 1 take a tile's two units. A tile's pages are asked for a tile
        // before they are needed.
        uint32_t ahead = x, left = 0, unit = 0, stop_unit = 0;  // the next item's place; tiles left of this one, this lane's unit, the end
        const uint8_t* head = nullptr;  // the head's first unit in page 0
        const int32_t* row = nullptr;   // the sequence's table
        int32_t page = 0;
        const uint32_t per = a.c.pshift - 4;
        auto look = [&]() {
            if (lane < 2 && unit < stop_unit) page = row[unit >> per];
        };
        auto enter = [&]() {  // the first tile from place `ahead` on
            while (ahead < end) {
                const Item it = item_at(ahead, end);
                const Entry& e = entries[it.entry];
                const uint32_t skip = it.place < START ? START - it.place : 0, here = it.stop - it.place;
                ahead = it.next;
                if (here <= skip || it.head0 + member >= a.c.heads) continue;
                left = here - skip;
                unit = e.unit0 + 2 * (it.place + skip - START) + lane;
                stop_unit = e.unit0 + e.units;
                row = a.c.table + static_cast<size_t>(e.seq) * a.c.max_pages;
                head = a.c.pages + a.layer * a.c.layer_bytes + (it.head0 + member) * a.c.head_bytes;
                look();
                break;
            }
        };
        auto fetch = [&](int stage) {
            if (!left) return;
            // of two units, the second may lie past the sequence's end (lane 0 knows)
            if (lane == 0) mbar_arrive_expect_tx(&full[warp][stage], (unit + 1 < stop_unit ? 2 : 1) * 18 * DK);
            __syncwarp();
            if (lane < 2 && unit < stop_unit) {
                if (page < 0 || static_cast<uint32_t>(page) >= a.c.n_pages) {
                    atomicOr(a.err, PKB_DEVERR_ARGS);  // any page will do, the rows are not defined
                    page = 0;
                }
                bulk_load(ring + (2 * stage + lane) * 18 * DK, head + static_cast<uint32_t>(page) * a.c.page_bytes + (unit & ((1u << per) - 1)) * (18 * DK),
                          18 * DK, &full[warp][stage]);
            }
            unit += 2;
            if (--left) look();
            else enter();
        };
        enter();
        int stage = 0, flying = 0;
        uint32_t phase = 0;
        bool lost = false;  // a wait ran out: the rest of the share is not computed
        for (; flying < STAGES && left; flying++) fetch(flying);
        while (x < end) {
            // one item, or the part of it in this share
            const Item it = item_at(x, end);
            const uint32_t x0 = x - it.place, stop = it.stop;
            x = it.next;
            const uint32_t h = it.head0 + member;
            if (stop <= START || h >= a.c.heads) continue;
            const Entry e = entries[it.entry];
            const uint32_t first = it.place < START ? 0 : it.place - START, block = it.block;
            Query<NB, NT, PARTS> q;
            load_query<T, NB, NT, PARTS>(a, e, h, block, q);
            int32_t all_lo = 0, all_hi = INT_MAX;  // the keys that every row of the block sees
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) {
                const Column c = column<NT>(a, e, block, i);
                if (c.valid) {
                    all_lo = max(all_lo, c.lo);
                    all_hi = min(all_hi, c.hi);
                }
            }
            all_lo = __reduce_max_sync(FULL, all_lo);
            all_hi = __reduce_min_sync(FULL, all_hi);
            float o[2 * NB][NT][4], m[2 * NT], l[2 * NT];
#pragma unroll
            for (int d = 0; d < 2 * NB; d++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int y = 0; y < 4; y++) o[d][j][y] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) m[i] = NEG_INF, l[i] = 0.0f;
            int32_t key0 = static_cast<int32_t>((e.unit0 + 2 * first) * C4_UNIT);
            for (uint32_t todo = lost ? 0 : stop - START - first; todo; todo--) {
                if (!warp_wait(&full[warp][stage], phase, &gave_up, a.timeout)) {
                    // a copy that does not come: say so, and let those in flight land
                    gave_up = 1;
                    if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
                    for (; flying; flying--) {
                        mbar_drain(&full[warp][stage], phase, a.timeout);
                        if (++stage == STAGES) stage = 0, phase ^= 1;
                    }
                    lost = true;
                    break;
                }
                uint8_t* buf = ring + stage * BYTES;
                // warp-uniform: tiles at the window's start, the causal edge and the last token
                const bool mask = key0 < all_lo || key0 + TILE > all_hi;
                tile_step<NB, NT, PARTS>(mask, a, e, block, buf, q, key0, static_cast<int32_t>(e.len), o, m, l);
                __syncwarp();
                if (left) fetch(stage);
                else flying--;  // nothing more to fetch: one copy fewer under way
                key0 += TILE;
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) l[i] = column_sum(l[i]);
            const bool entire = first == 0 && stop == it.places;
            if (entire && !lost) {
                write_rows<T, NB, NT>(a, e, h, block, o, l);
            } else if (!lost) {
                float4* part = reinterpret_cast<float4*>(a.part) + static_cast<size_t>(2 * v + (first == 0)) * (part_regs<NB, NT>() / 4) * 32 + lane;
#pragma unroll
                for (int d = 0; d < 2 * NB; d++)
#pragma unroll
                    for (int j = 0; j < NT; j++) part[(d * NT + j) * 32] = make_float4(o[d][j][0], o[d][j][1], o[d][j][2], o[d][j][3]);
#pragma unroll
                for (int j = 0; j < NT; j++) part[(NB * 2 * NT + j) * 32] = make_float4(m[2 * j], m[2 * j + 1], l[2 * j], l[2 * j + 1]);
            }
            // the share with an item's last tile says which shares have parts of
            // it, whatever became of them: the join reads what this call wrote alone
            if (stop == it.places && lane == 0) {
                const uint32_t team = it.head0 / a.team;
                a.joins[((static_cast<size_t>(it.entry) * a.teams + team) * a.max_blocks + block) * a.team + member] =
                    Attn4Join{entire || lost ? Attn4Join::NONE : split.of(x0 + START), share, e.r0, e.rows};
            }
        }
    }
    // blocks of rows that an entry does not have have nothing to join; entries that see no tokens are rows of zeros
    const uint32_t per_block = a.team, per_team = a.max_blocks * a.team;
    for (uint32_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        const Entry e = entries[i];
        const uint32_t blocks = base[i + 1] == base[i] ? 0 : e.blocks<NT>(a), none = (a.max_blocks - blocks) * per_block;
        for (uint32_t x = tid; x < a.teams * none; x += WORKERS * 32)
            a.joins[(static_cast<size_t>(i) * a.teams + x / none) * per_team + blocks * per_block + x % none].first = Attn4Join::NONE;
        if (blocks) continue;
        const uint32_t width = a.H * DK;
        for (uint64_t x = tid; x < static_cast<uint64_t>(e.rows) * width; x += WORKERS * 32)
            static_cast<T*>(a.o)[(e.r0 + x / width) * a.os + x % width] = c4_round<T>(0.0f);
    }
}

// Joins the parts of the items that several shares have. A warp takes 16
// dimensions of eight rows (a float4 a lane) over every `ways`-th of an
// item's parts; `ways` warps then join theirs, always in the same order. It
// is bound by latency: the item, then its parts, one load behind the other.
// Up to eight parts an item go one way (a step of 32 sequences of 400 tokens, 16
// heads, five parts each: 20.1 us with its join, 21.5 two ways; 8 heads, nine parts
// each: 17.5, 15.8 two ways), a few long items' take up to eight, so that no
// warp reads many parts one after another (three sequences of up to 120,001 tokens 62.7
// us, 72.5 two ways). Four parts are loaded together (in 64 registers, so that
// four blocks share an SM), or eight where each way still has more than six (the same three
// 65.6 -> 62.7 us; 8 of 400 tokens, five parts a way, 12.8 and 15.0 with eight, in graphs).
template <typename T, int NB, int NT, int BATCH>
__global__ void __launch_bounds__(JOIN_WARPS * 32, BATCH == 4 ? 4 : 2) join_kernel(Attn4Args a, uint32_t ways) {
    constexpr int QUADS = 2 * NB * NT, STRIDE = part_regs<NB, NT>() / 4;  // float4s of a lane: [dims 16][eight rows], then m and l
    __shared__ float4 sm[2][JOIN_WARPS][32];
    pdl_trigger();
    pdl_wait();
    // the item: [entry][team][block][member]
    const uint32_t member = blockIdx.x % a.team, block = blockIdx.x / a.team % a.max_blocks, h = blockIdx.x / a.team / a.max_blocks % a.teams * a.team + member;
    if (h >= a.c.heads) return;
    const Attn4Join item = a.joins[blockIdx.x];
    if (item.first == Attn4Join::NONE) return;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, warp = threadIdx.x / 32, way = warp % ways;
    const uint32_t z = blockIdx.y * (JOIN_WARPS / ways) + warp / ways;
    const uint32_t d = z / NT, j = z % NT;
    float m0 = NEG_INF, m1 = NEG_INF, l0 = 0.0f, l1 = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t all = item.last - item.first + 1, count = all > way ? (all - way + ways - 1) / ways : 0;
    if (z < QUADS) {
        const float4* part = reinterpret_cast<const float4*>(a.part) + lane;
        // all of a batch's loads before the first use
        for (uint32_t i0 = 0; i0 < count; i0 += BATCH) {
            float4 v[BATCH], x[BATCH];
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                v[i] = make_float4(NEG_INF, NEG_INF, 0.0f, 0.0f);
                x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i0 + i < count) {
                    const uint32_t s = item.first + way + (i0 + i) * ways;
                    const float4* p = part + static_cast<size_t>(2 * (s * a.team + member) + (s == item.first)) * STRIDE * 32;
                    v[i] = p[(QUADS + j) * 32];
                    x[i] = p[z * 32];
                }
            }
            float t0 = m0, t1 = m1;
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                t0 = fmaxf(t0, v[i].x);
                t1 = fmaxf(t1, v[i].y);
            }
            const float k0 = rescale(m0, t0), k1 = rescale(m1, t1);
            m0 = t0, m1 = t1;
            l0 *= k0, l1 *= k1, o[0] *= k0, o[1] *= k1, o[2] *= k0, o[3] *= k1;
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                const float f0 = rescale(v[i].x, m0), f1 = rescale(v[i].y, m1);
                l0 = __fmaf_rn(v[i].z, f0, l0);
                l1 = __fmaf_rn(v[i].w, f1, l1);
                o[0] = __fmaf_rn(x[i].x, f0, o[0]);
                o[1] = __fmaf_rn(x[i].y, f1, o[1]);
                o[2] = __fmaf_rn(x[i].z, f0, o[2]);
                o[3] = __fmaf_rn(x[i].w, f1, o[3]);
            }
        }
    }
    if (ways > 1) {
        sm[0][warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
        sm[1][warp][lane] = make_float4(m0, m1, l0, l1);
        __syncthreads();
        if (way) return;
        for (uint32_t w = 1; w < ways; w++) {
            const float4 v = sm[1][warp + w][lane], x = sm[0][warp + w][lane];
            const float t0 = fmaxf(m0, v.x), t1 = fmaxf(m1, v.y);
            const float k0 = rescale(m0, t0), k1 = rescale(m1, t1), f0 = rescale(v.x, t0), f1 = rescale(v.y, t1);
            m0 = t0, m1 = t1;
            l0 = l0 * k0 + v.z * f0;
            l1 = l1 * k1 + v.w * f1;
            o[0] = o[0] * k0 + x.x * f0;
            o[1] = o[1] * k1 + x.y * f1;
            o[2] = o[2] * k0 + x.z * f0;
            o[3] = o[3] * k1 + x.w * f1;
        }
    }
    if (z >= QUADS) return;
    const Entry e = {0, item.r0, item.rows, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const Column c = column<NT>(a, e, block, 2 * j + i);
        if (!c.valid) continue;
        const float l = i ? l1 : l0, inv = l == 0.0f ? 0.0f : __fdiv_rn(4.0f, l);
        T* out = static_cast<T*>(a.o) + static_cast<size_t>(e.r0 + c.tok) * a.os + (h * a.G + c.r - c.tok * a.G) * (NB * 32) + d * 16 + g;
        out[0] = c4_round<T>(__fmul_rn(o[i], inv));
        out[8] = c4_round<T>(__fmul_rn(o[2 + i], inv));
    }
}

// ---------------------------------------------------------- many rows --
//
// Prompts and long chunks: a block takes ROW_WARPS blocks of rows of one
// entry and head, a warp each, and its warps read the same tiles from one
// ring, so that a tile is fetched once for 64 or 128 rows. Nothing is split
// along the keys. A warp leaves out the tiles that its own rows cannot see.
// For f16 and float rows, and bf16 rows of 256 values (others: pkb_attn4_tc.cu).
// Bound by the tile's instructions and mma.sync's rate: 3 (f16 and bf16) or 5
// (float rows) products of 16 keys and 8 rows a 16 values. 8 sequences of 2,048
// tokens, 8 heads of 128, 256 float rows a head: 193 us.

constexpr int ROW_WARPS = 8;
constexpr int ROW_STAGES = 8;

template <typename T, int NB, int NT, int PARTS>
__global__ void __launch_bounds__((ROW_WARPS + 1) * 32, 1) rows_kernel(Attn4Args a) {
    constexpr int DK = NB * 32, BYTES = tile_bytes<NB>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[ROW_STAGES], empty[ROW_STAGES];
    __shared__ volatile int gave_up;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (tid == 0) {
        for (int i = 0; i < ROW_STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], ROW_WARPS);
        }
        fence_mbar_init();
        gave_up = 0;
    }
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    const uint32_t h = blockIdx.y;
    const Entry e = load_entry(a, blockIdx.z);
    // the last rows, which see most, begin first
    const uint32_t groups = (e.blocks<NT>(a) + ROW_WARPS - 1) / ROW_WARPS;
    if (blockIdx.x >= groups) return;
    const uint32_t group = groups - 1 - blockIdx.x, block = group * ROW_WARPS + warp;
    // the units that the block's rows can see
    const uint32_t tok0 = group * ROW_WARPS * 8 * NT / a.G, tok1 = min((group + 1) * ROW_WARPS * 8 * NT - 1, e.rows * a.G - 1) / a.G;
    const int32_t lo = keys_of(a, e, tok0).lo, hi = keys_of(a, e, tok1).hi;
    const uint32_t unit0 = static_cast<uint32_t>(lo / C4_UNIT);
    const uint32_t units = hi > lo ? static_cast<uint32_t>((hi + C4_UNIT - 1) / C4_UNIT) - unit0 : 0, tiles = (units + 1) / 2;

    if (warp == ROW_WARPS) {
        const uint32_t per = a.c.pshift - 4;
        const int32_t* row = a.c.table + static_cast<size_t>(e.seq) * a.c.max_pages;
        const uint8_t* head = a.c.pages + a.layer * a.c.layer_bytes + h * a.c.head_bytes;
        int32_t page = lane < 2 && lane < units ? row[(unit0 + lane) >> per] : 0;
        uint32_t issued = 0;
        for (uint32_t i = 0; i < tiles; i++, issued++) {
            const int stage = i % ROW_STAGES;
            if (!warp_wait(&empty[stage], (i / ROW_STAGES & 1) ^ 1, &gave_up, a.timeout)) {
                gave_up = 1;
                if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
                break;
            }
            const uint32_t unit = unit0 + 2 * i + lane;
            if (lane == 0) mbar_arrive_expect_tx(&full[stage], (units - 2 * i < 2 ? 1 : 2) * 18 * DK);
            __syncwarp();
            if (lane < 2 && 2 * i + lane < units) {
                if (page < 0 || static_cast<uint32_t>(page) >= a.c.n_pages) {
                    atomicOr(a.err, PKB_DEVERR_ARGS);  // any page will do, the rows are not defined
                    page = 0;
                }
                bulk_load(smem + stage * BYTES + lane * 18 * DK, head + static_cast<uint32_t>(page) * a.c.page_bytes + (unit & ((1u << per) - 1)) * (18 * DK),
                          18 * DK, &full[stage]);
                if (2 * i + 2 + lane < units) page = row[(unit + 2) >> per];
            }
        }
        // whatever the others did, the copies in flight land before the block leaves its memory
        for (uint32_t i = issued < ROW_STAGES ? 0 : issued - ROW_STAGES; i < issued; i++)
            mbar_drain(&full[i % ROW_STAGES], i / ROW_STAGES & 1, a.timeout);
        return;
    }

    Query<NB, NT, PARTS> q;
    load_query<T, NB, NT, PARTS>(a, e, h, block, q);
    int32_t all_lo = 0, all_hi = INT_MAX, any_lo = INT_MAX, any_hi = 0;  // the keys that every row, and that any row of the warp sees
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
        const Column c = column<NT>(a, e, block, i);
        if (c.valid) {
            all_lo = max(all_lo, c.lo);
            all_hi = min(all_hi, c.hi);
            any_lo = min(any_lo, c.lo);
            any_hi = max(any_hi, c.hi);
        }
    }
    all_lo = __reduce_max_sync(FULL, all_lo);
    all_hi = __reduce_min_sync(FULL, all_hi);
    any_lo = __reduce_min_sync(FULL, any_lo);
    any_hi = __reduce_max_sync(FULL, any_hi);
    float o[2 * NB][NT][4], m[2 * NT], l[2 * NT];
#pragma unroll
    for (int d = 0; d < 2 * NB; d++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int y = 0; y < 4; y++) o[d][j][y] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) m[i] = NEG_INF, l[i] = 0.0f;
    int32_t key0 = static_cast<int32_t>(unit0 * C4_UNIT);
    for (uint32_t i = 0; i < tiles; i++, key0 += TILE) {
        const int stage = i % ROW_STAGES;
        if (!warp_wait(&full[stage], i / ROW_STAGES & 1, &gave_up, a.timeout)) {
            gave_up = 1;  // the producer lets what is in flight land
            if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
            return;
        }
        if (key0 < any_hi && key0 + TILE > any_lo) {
            const bool mask = key0 < all_lo || key0 + TILE > all_hi;
            tile_step<NB, NT, PARTS>(mask, a, e, block, smem + stage * BYTES, q, key0, hi, o, m, l);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
    }
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) l[i] = column_sum(l[i]);
    write_rows<T, NB, NT>(a, e, h, block, o, l);
}

// ------------------------------------------------------------------- host --

template <int NB, int NT> size_t split_smem(uint32_t n) {
    return workers<NB, NT>() * stages<NB, NT>() * tile_bytes<NB>() + static_cast<size_t>(n) * (sizeof(Entry) + 4) + 4;
}

// What attention4_tc_takes leaves to rows_kernel: the others are not built.
template <typename T, int NB> constexpr bool has_rows_kernel() { return !std::is_same<T, __nv_bfloat16>::value || NB == 8; }

template <typename T, int NB, int NT, int PARTS>
cudaError_t prepare_one() {
    if constexpr (has_rows_kernel<T, NB>()) {
        const cudaError_t e = cudaFuncSetAttribute(rows_kernel<T, NB, NT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   ROW_STAGES * tile_bytes<NB>());
        if (e != cudaSuccess) return e;
    }
    return cudaFuncSetAttribute(split_kernel<T, NB, NT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(split_smem<NB, NT>(MAX_ENTRIES)));
}

template <typename T, int PARTS>
cudaError_t prepare_type() {
    cudaError_t e;
    if ((e = prepare_one<T, 1, 1, PARTS>()) || (e = prepare_one<T, 1, 2, PARTS>()) || (e = prepare_one<T, 2, 1, PARTS>()) ||
        (e = prepare_one<T, 2, 2, PARTS>()) || (e = prepare_one<T, 3, 1, PARTS>()) || (e = prepare_one<T, 3, 2, PARTS>()) ||
        (e = prepare_one<T, 4, 1, PARTS>()) || (e = prepare_one<T, 4, 2, PARTS>()) || (e = prepare_one<T, 8, 1, PARTS>()))
        return e;
    return cudaSuccess;
}

template <typename T, int NB, int NT, int PARTS>
cudaError_t launch_rows(const Attn4Args& a, cudaStream_t s) {
    const uint32_t most = ROW_WARPS * 8 * NT;
    const dim3 grid((a.max_rows * a.G + most - 1) / most, a.c.heads, a.n);
    const cudaError_t e = c4_launch(rows_kernel<T, NB, NT, PARTS>, grid, (ROW_WARPS + 1) * 32, ROW_STAGES * tile_bytes<NB>(), s, a);
    if (e == cudaSuccess) count_launch();
    return e;
}

template <typename T, int NB, int NT, int PARTS>
cudaError_t launch_split(Attn4Args a, uint32_t grid, cudaStream_t s) {
    a.max_blocks = (a.max_rows * a.G + 8 * NT - 1) / (8 * NT);
    cudaError_t e = c4_launch(split_kernel<T, NB, NT, PARTS>, grid, workers<NB, NT>() * 32, split_smem<NB, NT>(a.n), s, a);
    if (e != cudaSuccess) return e;
    count_launch();
    // Parts an item has about, if all have as many: more than eight go two ways
    // and so on, more than 48 eight at a time.
    const uint64_t items = static_cast<uint64_t>(a.n) * a.teams * a.max_blocks, most = grid * workers<NB, NT>() / a.team;
    const uint64_t shares = most < a.max_shares ? most : a.max_shares;
    uint32_t ways = 1;
    while (ways < 8 && shares > 8 * ways * items) ways *= 2;
    const uint32_t quads = JOIN_WARPS / ways;
    e = c4_launch(shares > 48 * items ? join_kernel<T, NB, NT, 8> : join_kernel<T, NB, NT, 4>,
                  dim3(static_cast<uint32_t>(items * a.team), (2 * NB * NT + quads - 1) / quads), JOIN_WARPS * 32, 0, s, a, ways);
    if (e == cudaSuccess) count_launch();
    return e;
}

template <typename T, int NB, int NT, int PARTS>
cudaError_t launch_one(const Attn4Args& a, uint32_t grid, bool split, cudaStream_t s) {
    if (split) return launch_split<T, NB, NT, PARTS>(a, grid, s);
    if constexpr (has_rows_kernel<T, NB>()) return launch_rows<T, NB, NT, PARTS>(a, s);
    return cudaErrorInvalidValue;
}

// Rows of a block: two blocks of eight share the codes' conversion where there
// are more than eight rows (64 sequences of 2,048 tokens, heads of 128, bf16: 16
// rows 72 us, 88 in eights; 4 rows 71, 52 in eights). Half of the last sixteen
// is empty for 17 to 24 rows, which are three eights (32 sequences of 1,500
// tokens: f16 54 us, 55.5 in sixteens; float 67 and 74.5), and for 33 to 40, which are five where they
// are float, whose five products a 16 values are most of the work (103 us, 107 in
// sixteens; f16 82.6 and 78); 52 rows are better off in sixteens (float 163 and 143).
uint32_t block_rows(const Attn4Args& a, bool float_rows) {
    const uint64_t rows = static_cast<uint64_t>(a.max_rows) * a.G, eights = (rows + 7) / 8;
    return a.c.dk == 256 || eights == 1 || eights == 3 || (eights == 5 && float_rows) ? 8 : 16;
}

template <typename T, int PARTS>
cudaError_t launch_type(const Attn4Args& a, uint32_t grid, bool split, cudaStream_t s) {
    const bool two = block_rows(a, PARTS == 3) == 16;
    switch (a.c.dk) {
        case 32: return two ? launch_one<T, 1, 2, PARTS>(a, grid, split, s) : launch_one<T, 1, 1, PARTS>(a, grid, split, s);
        case 64: return two ? launch_one<T, 2, 2, PARTS>(a, grid, split, s) : launch_one<T, 2, 1, PARTS>(a, grid, split, s);
        case 96: return two ? launch_one<T, 3, 2, PARTS>(a, grid, split, s) : launch_one<T, 3, 1, PARTS>(a, grid, split, s);
        case 128: return two ? launch_one<T, 4, 2, PARTS>(a, grid, split, s) : launch_one<T, 4, 1, PARTS>(a, grid, split, s);
        default: return launch_one<T, 8, 1, PARTS>(a, grid, split, s);
    }
}

bool is_aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Cached heads as teams of at most MAX_TEAM, of one size but for the last.
void teams_of(uint32_t heads, uint32_t* team, uint32_t* teams) {
    *teams = (heads + MAX_TEAM - 1) / MAX_TEAM;
    *team = (heads + *teams - 1) / *teams;
}

// Places of a sequence at most, whatever its length: they are counted in 32 bits.
uint64_t places_of(const pkb_cache4* c) { return static_cast<uint64_t>(c->max_pages) * c->page_tokens / TILE + 1 + START; }

// Whether `rows` rows of each of n entries are split along the keys, or taken
// by blocks that go over all of an entry's keys. Lengths are not known here,
// but both ways' times are proportional to them, so only the grids count:
//  - bf16 on tcgen05: 16 rows of a split take the GPU as long as half an SM
//    takes to do 256, or, where those are one tile of 128 and of heads so wide
//    that unpacking bounds the split, as two thirds of one take (8 sequences of 2,048 tokens, 8 heads of 128
//    with 4 query heads each: 16 tokens 41 us split and 33 so, heads of 64 28.5
//    and 29.5; 2 sequences of 4,096, 64 tokens: 68 and 77; one of 8,192: 67 and 142).
//  - others: rows_kernel's warps are as fast as the split's, and leave out what
//    a prompt's rows cannot see, half of it at most: it is worth an
//    SM's eight warps where half of all SMs' have work (float rows of 24
//    sequences of 600 tokens, 100 tokens each: 106 us split and 117 so; of one
//    sequence of 8,192, 64 tokens with 4 query heads each: 89 and 735).
bool splits(const Attn4Args& a, int type, uint32_t n, uint32_t grid) {
    const uint64_t rows = static_cast<uint64_t>(a.max_rows) * a.G, heads = static_cast<uint64_t>(n) * a.teams * a.team;
    if (rows > SPLIT_ROWS) return false;
    const bool tc = attention4_tc_takes(a, type);
    if (!tc && rows <= 128) return true;
    const uint64_t block = tc ? 16 : block_rows(a, type == PKB_F32), blocks = (rows + block - 1) / block;
    const uint64_t many = tc ? 256 : ROW_WARPS * block, waves = (heads * ((rows + many - 1) / many) + grid - 1) / grid;
    return 2 * heads * blocks <= (!tc ? 8 : rows <= 128 && a.c.dk >= 96 ? 3 : 4) * grid * waves;
}

// The work area of a call, over any lengths and max_rows: a join an item (an
// entry, head and block of rows), two parts a share and head. Up to 128 rows
// are 16 blocks at most. More are nine or more, and `splits` wants them to be
// at most 4 (blocks / 8, rounded up) a head and 4 grids beside, so that heads times
// blocks stay within 36 grids (nine blocks; fewer for others and on tcgen05's side).
struct Bounds {
    uint64_t shares, join_bytes, bytes;
};

Bounds bounds_of(const pkb_cache4* c, uint32_t H, uint32_t rows, uint32_t n) {
    uint32_t team, teams;
    teams_of(c->n_heads, &team, &teams);
    const uint64_t all = static_cast<uint64_t>(rows) * (H / c->n_heads), blocks = all < 128 ? (all + 7) / 8 : 16;
    uint64_t items = static_cast<uint64_t>(n < MAX_ENTRIES ? n : MAX_ENTRIES) * teams * team * blocks;
    if (all > 128 && items < 36 * MAX_GRID) items = 36 * MAX_GRID;
    const uint64_t most = static_cast<uint64_t>(MAX_GRID) * MAX_WORKERS / team, places = items / team * places_of(c);
    Bounds b;
    b.shares = places < most ? places : most;
    b.join_bytes = (items * sizeof(Attn4Join) + 255) & ~static_cast<uint64_t>(255);
    b.bytes = b.join_bytes + 2 * b.shares * team * (c->head_dim == 256 ? 1 : 2) * (c->head_dim / 4 + 4) * 128;
    return b;
}

// The kernels' attributes, at the first call on a device: it loads them all,
// some 15 ms that a program without a cache does not pay at its own first call.
constexpr int MAX_DEV = 16;  // current_device_info has checked that the device is below it
std::mutex g_mu;
std::atomic<bool> g_ready[MAX_DEV];

cudaError_t prepare() {
    int dev;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || g_ready[dev].load(std::memory_order_acquire)) return e;
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_ready[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = prepare_type<float, 3>();
    if (e == cudaSuccess) e = prepare_type<__half, 2>();
    if (e == cudaSuccess) e = prepare_type<__nv_bfloat16, 2>();
    if (e == cudaSuccess) e = prepare_attention4_tc();
    if (e == cudaSuccess) g_ready[dev].store(true, std::memory_order_release);
    return e;
}

}  // namespace

}  // namespace pkb

using namespace pkb;

extern "C" {

size_t pkb_attention_cache4_work_bytes(const pkb_cache4* c, uint32_t H, uint32_t rows, uint32_t n) {
    if (!c || !pkb_cache4_page_bytes(c->page_tokens, c->n_heads, c->head_dim) || !H || H % c->n_heads) return 0;
    return rows && n ? bounds_of(c, H, rows, n).bytes : 0;
}

int pkb_attention_cache4_dev(void* stream, void* o, size_t os, const void* q, size_t qs, int type, uint32_t H,
                             const pkb_cache4* c, uint32_t layer, const int32_t* seqs, const int32_t* starts,
                             uint32_t n, uint32_t rows, uint32_t max_rows, float scale, int causal, uint32_t window,
                             void* work, size_t work_bytes) {
    const char* who = "attention_cache4";
    Attn4Args a = {};
    int rc = c4_view(c, who, &a.c);
    if (rc) return rc;
    if ((rc = c4_check_type(type, who))) return rc;
    if (layer >= c->n_layers) return set_error(PKB_EINVAL, "%s: layer %u of %u", who, layer, c->n_layers);
    if (!H || H % c->n_heads) return set_error(PKB_EINVAL, "%s: H = %u, a multiple of the cache's %u heads", who, H, c->n_heads);
    a.scale = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634074);  // log2 e
    if (!(a.scale - a.scale == 0.0f)) return set_error(PKB_EINVAL, "%s: scale log2 e is not finite", who);
    if (window > INT_MAX) return set_error(PKB_EINVAL, "%s: window = %u", who, window);
    // one that reaches past every sequence's first token from its last row on is none
    if (window >= static_cast<uint64_t>(c->max_pages) * c->page_tokens + max_rows) window = 0;
    if (!n || !rows) return PKB_OK;
    if (n > INT_MAX) return set_error(PKB_EINVAL, "%s: %u sequences", who, n);
    if (!o || !q || !seqs || !starts || !work) return set_error(PKB_EINVAL, "%s: null pointer", who);
    if (!max_rows || max_rows > rows) return set_error(PKB_EINVAL, "%s: max_rows = %u of %u rows", who, max_rows, rows);
    const size_t width = static_cast<size_t>(H) * c->head_dim, size = c4_type_bytes(type);
    if (width > UINT_MAX / 2 || rows > INT_MAX || static_cast<uint64_t>(rows) * (H / c->n_heads) > INT_MAX) return set_error(PKB_EINVAL, "%s: %u rows of %zu values", who, rows, width);
    if (rows > 1 && (qs < width || os < width)) return set_error(PKB_EINVAL, "%s: a row stride below %zu values", who, width);
    if (rows == 1) qs = os = width;
    if (!is_aligned(o, size) || !is_aligned(q, size) || !is_aligned(seqs, 4) || !is_aligned(starts, 4))
        return set_error(PKB_EINVAL, "%s: misaligned buffer", who);
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), q1 = q0 + ((rows - 1) * qs + width) * size;
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(o), o1 = o0 + ((rows - 1) * os + width) * size;
    if (o0 < q1 && q0 < o1) return set_error(PKB_EINVAL, "%s: o overlaps q", who);
    const Bounds bounds = bounds_of(c, H, rows, n);
    if (work_bytes < bounds.bytes || !is_aligned(work, 256))
        return set_error(PKB_EINVAL, "%s: work area of %zu bytes (%zu needed, 256-byte aligned)", who, work_bytes, static_cast<size_t>(bounds.bytes));
    int sms;
    if ((rc = current_device_info(&sms, &a.err))) return rc;
    const cudaError_t set_up = prepare();
    if (set_up != cudaSuccess) return set_error(PKB_ECUDA, "%s kernel attributes: %s", who, cudaGetErrorString(set_up));
    a.q = q;
    a.o = o;
    a.qs = qs;
    a.os = os;
    a.layer = layer;
    a.rows = rows;
    a.H = H;
    a.G = H / c->n_heads;
    a.vec = is_aligned(q, 16) && qs * size % 16 == 0;
    a.vec_o = is_aligned(o, 16) && os * size % 16 == 0;
    a.causal = causal ? 1 : 0;
    a.window = window;
    a.timeout = wait_cycles();
    a.max_rows = max_rows;
    teams_of(c->n_heads, &a.team, &a.teams);
    a.joins = static_cast<Attn4Join*>(work);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + bounds.join_bytes);
    a.max_shares = static_cast<uint32_t>(bounds.shares);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint32_t grid = static_cast<uint32_t>(sms < MAX_GRID ? sms : MAX_GRID);
    // entries of a launch: a split's places are counted in 32 bits
    const uint64_t entry = places_of(c) * a.teams * ((static_cast<uint64_t>(max_rows) * a.G + 7) / 8);
    const bool split = splits(a, type, n, grid) && entry <= UINT_MAX;
    const uint32_t step = split && UINT_MAX / entry < MAX_ENTRIES ? static_cast<uint32_t>(UINT_MAX / entry) : MAX_ENTRIES;
    for (uint32_t i = 0; i < n; i += step) {
        a.seqs = seqs + i;
        a.starts = starts + i;
        a.n = n - i < step ? n - i : step;
        const cudaError_t e = !split && attention4_tc_takes(a, type) ? launch_attention4_tc(a, s)
                              : type == PKB_F32 ? launch_type<float, 3>(a, grid, split, s)
                              : type == PKB_F16 ? launch_type<__half, 2>(a, grid, split, s)
                                                : launch_type<__nv_bfloat16, 2>(a, grid, split, s);
        if (e != cudaSuccess)
            return set_error(e == cudaErrorMemoryAllocation ? PKB_ENOMEM : PKB_ECUDA, "%s launch: %s", who, cudaGetErrorString(e));
    }
    return PKB_OK;
}

}  // extern "C"
