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
// no value crosses a lane.
//
// The split. All (sequence, head, block of rows) items' tiles of 32 keys are
// laid end to end and divided evenly over all warps of the GPU, whatever
// the sequences' lengths: a warp's share begins and ends inside items. A warp
// streams its tiles through a ring of its own in shared memory (bulk
// copies of whole units, 18 dk bytes, completing on its mbarriers), so warps
// never wait for one another. An item that one warp has whole is written
// at once; of the others each warp leaves its part (m, l, O) in the work
// area, and a second kernel joins an item's parts in a fixed order.

#include <climits>

#include "pkb_attn4.cuh"
#include "pkb_internal.h"

namespace pkb {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int WARPS = 8;
constexpr int TILE = 32;            // keys of a tile: two units
constexpr uint32_t MAX_ENTRIES = 1024;  // sequences of one launch
constexpr int MAX_GRID = 320;
constexpr uint64_t MIN_TILES = 2;   // of a warp's share, where there are so many

template <int NB> __host__ __device__ constexpr int stages() { return NB <= 2 ? 4 : NB == 3 ? 3 : 2; }
template <int NB> __host__ __device__ constexpr int tile_bytes() { return 2 * 18 * 32 * NB; }
template <int NB, int NT> __host__ __device__ constexpr int part_regs() { return NT * (NB * 8 + 4); }  // a lane's of one part
template <int NB, int NT, int PARTS> constexpr int blocks_per_sm() { return NB * 8 * NT + NB * 4 * NT * PARTS <= 80 && NB <= 4 ? 2 : 1; }

// One entry's shape: its rows, tokens, and the units its rows can see.
struct Entry {
    uint32_t seq, r0, rows, len, unit0, units, tiles, blocks;
};

template <int NT>
__device__ __forceinline__ Entry load_entry(const Attn4Args& a, uint32_t i) {
    Entry e;
    e.rows = c4_rows(a.c, a.seqs, a.starts, i, a.rows, &e.seq, &e.r0, a.err);
    e.len = e.rows ? c4_len(a.c, e.seq, a.err) : 0;
    // the first row's window begins furthest back; the last row's causal end is len
    const int64_t lo = a.window ? static_cast<int64_t>(e.len) - e.rows - a.window + 1 : 0;
    e.unit0 = lo > 0 ? static_cast<uint32_t>(lo) / C4_UNIT : 0;
    e.units = (e.len + C4_UNIT - 1) / C4_UNIT - e.unit0;
    e.tiles = (e.units + 1) / 2;
    e.blocks = static_cast<uint32_t>((static_cast<uint64_t>(e.rows) * a.G + 8 * NT - 1) / (8 * NT));
    return e;
}

// how many warps share `total` tiles, and where warp w's share begins
__device__ __forceinline__ uint64_t shares(const Attn4Args& a, uint64_t total, uint64_t warps) {
    const uint64_t most = (total + MIN_TILES - 1) / MIN_TILES, room = warps < a.max_shares ? warps : a.max_shares;
    return most < room ? most : room;
}
__device__ __forceinline__ uint64_t share_begin(uint64_t w, uint64_t total, uint64_t n) { return w * total / n; }

// A lane's two columns of each eight rows: where they end up and what they
// may see.
template <int NT>
struct Columns {
    int64_t row[2 * NT];  // of o, -1: none
    uint32_t head[2 * NT];
    int32_t lo[2 * NT], hi[2 * NT];  // keys [lo, hi)
};

template <int NT>
__device__ __forceinline__ void load_columns(const Attn4Args& a, const Entry& e, uint32_t h, uint32_t block, Columns<NT>& col) {
    const uint32_t t = threadIdx.x & 3;
    const uint64_t all = static_cast<uint64_t>(e.rows) * a.G;
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
        const uint64_t r = static_cast<uint64_t>(block) * (8 * NT) + i / 2 * 8 + 2 * t + i % 2;
        const uint64_t tok = r / a.G;
        const int64_t pos = static_cast<int64_t>(e.len) - e.rows + static_cast<int64_t>(tok);
        const int64_t hi = a.causal ? pos + 1 : e.len, lo = a.window ? pos - a.window + 1 : 0;
        col.row[i] = r < all ? static_cast<int64_t>(e.r0 + tok) : -1;
        col.head[i] = h * a.G + static_cast<uint32_t>(r % a.G);
        col.hi[i] = r < all ? static_cast<int32_t>(hi < 0 ? 0 : hi > e.len ? e.len : hi) : 0;
        col.lo[i] = static_cast<int32_t>(lo < 0 ? 0 : lo > INT_MAX ? INT_MAX : lo);
    }
}

template <typename T, int NB, int NT>
__device__ __forceinline__ void write_rows(const Attn4Args& a, const Columns<NT>& col, const float (&o)[2 * NB][NT][4],
                                           const float (&l)[2 * NT]) {
    const uint32_t g = (threadIdx.x & 31) / 4;
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
        if (col.row[i] < 0) continue;
        T* out = static_cast<T*>(a.o) + col.row[i] * a.os + static_cast<size_t>(col.head[i]) * (NB * 32) + g;
        // a row that sees nothing has sum 0 and is zeros; a NaN sum gives NaNs
        const float inv = l[i] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[i]);
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

// One tile of two units at `buf`: its scores, the softmax's step, its values.
// MASK: some key of it is hidden from some row, or lies past the last token.
template <int NB, int NT, int PARTS, bool MASK>
__device__ __forceinline__ void tile_step(const uint8_t* buf, const uint32_t (&q)[NB][2][NT][PARTS][2], const Columns<NT>& col,
                                          int32_t key0, int32_t len, float scale, float (&o)[2 * NB][NT][4], float (&m)[2 * NT],
                                          float (&l)[2 * NT]) {
    constexpr int DK = NB * 32;
    const uint32_t lane = threadIdx.x & 31, g = lane / 4, t = lane & 3;
    float s[2][NT][4];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const uint8_t* unit = buf + u * 18 * DK;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int x = 0; x < 4; x++) s[u][j][x] = 0.0f;
        uint32_t w[2][NB];
        lds_words<NB>(unit + (g * 4 + t) * NB * 4, w[0]);
        lds_words<NB>(unit + ((g + 8) * 4 + t) * NB * 4, w[1]);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t s2[2], ms[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint32_t half = *reinterpret_cast<const uint16_t*>(unit + 16 * DK + ((g + 8 * r) * NB + b) * 2);
                s2[r] = half | half << 16;
                ms[r] = c4_m24(s2[r]);
            }
            float fresh[NT][4];
            if constexpr (PARTS == 3) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) fresh[j][x] = 0.0f;
            }
#pragma unroll
            for (int step = 0; step < 2; step++) {
                uint32_t a[4];
                if (step == 0) {
                    a[0] = c4_pair<0>(w[0][b], s2[0], ms[0]);
                    a[1] = c4_pair<0>(w[1][b], s2[1], ms[1]);
                    a[2] = c4_pair<1>(w[0][b], s2[0], ms[0]);
                    a[3] = c4_pair<1>(w[1][b], s2[1], ms[1]);
                } else {
                    a[0] = c4_pair<2>(w[0][b], s2[0], ms[0]);
                    a[1] = c4_pair<2>(w[1][b], s2[1], ms[1]);
                    a[2] = c4_pair<3>(w[0][b], s2[0], ms[0]);
                    a[3] = c4_pair<3>(w[1][b], s2[1], ms[1]);
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; p--)
                        mma_bf16(PARTS == 3 ? fresh[j] : s[u][j], a, q[b][step][j][p][0], q[b][step][j][p][1]);
            }
            // the tensor cores cut what they add; for float rows each
            // block's sum is added by a rounded addition instead
            if constexpr (PARTS == 3) {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[u][j][x] = __fadd_rn(s[u][j][x], fresh[j][x]);
            }
        }
    }
    bool above = false;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                float y = __fmul_rn(s[u][j][x], scale);
                const int i = 2 * j + (x & 1);
                if constexpr (MASK) {
                    const int32_t key = key0 + 16 * u + static_cast<int32_t>(g) + 8 * (x / 2);
                    y = key >= col.lo[i] && key < col.hi[i] ? y : NEG_INF;
                }
                above |= y > m[i] + 8.0f;
                s[u][j][x] = y;
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
                if constexpr (MASK) {  // scales past the last token may be anything, and 0 times a NaN is one
                    const int32_t key = key0 + 16 * u + 8 * c + 2 * static_cast<int32_t>(t);
                    if (key >= len) s2[c] = 0;
                    else if (key + 1 >= len) s2[c] &= 0xFFFFu;
                }
                ms[c] = c4_m24(s2[c]);
            }
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const uint32_t x = d ? w.y : w.x;
                uint32_t a[4];
                a[0] = c4_pair<0>(x, s2[0], ms[0]);
                a[1] = c4_pair<1>(x, s2[0], ms[0]);
                a[2] = c4_pair<2>(x, s2[1], ms[1]);
                a[3] = c4_pair<3>(x, s2[1], ms[1]);
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
__global__ void __launch_bounds__(WARPS * 32, blocks_per_sm<NB, NT, PARTS>()) split_kernel(Attn4Args a) {
    constexpr int DK = NB * 32, STAGES = stages<NB>(), BYTES = tile_bytes<NB>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[WARPS][STAGES];
    __shared__ uint64_t sums[WARPS];
    __shared__ volatile int gave_up;
    uint64_t* base = reinterpret_cast<uint64_t*>(smem + WARPS * STAGES * BYTES);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (lane == 0) {
        for (int i = 0; i < STAGES; i++) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }
    if (tid == 0) gave_up = 0;
    pdl_trigger();
    pdl_wait();
    // each entry's first tile: four entries a thread, a scan over the block
    uint64_t mine[MAX_ENTRIES / (WARPS * 32)], own = 0;
#pragma unroll
    for (int x = 0; x < static_cast<int>(MAX_ENTRIES / (WARPS * 32)); x++) {
        const uint32_t i = tid * (MAX_ENTRIES / (WARPS * 32)) + x;
        mine[x] = own;
        if (i < a.n) {
            const Entry e = load_entry<NT>(a, i);
            own += static_cast<uint64_t>(e.tiles) * a.c.heads * e.blocks;
        }
    }
    uint64_t scan = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint64_t y = __shfl_up_sync(FULL, scan, d);
        if (lane >= static_cast<uint32_t>(d)) scan += y;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t w = 0; w < WARPS; w++) {
        if (w == warp) scan += total - own;
        total += sums[w];
    }
#pragma unroll
    for (int x = 0; x < static_cast<int>(MAX_ENTRIES / (WARPS * 32)); x++) {
        const uint32_t i = tid * (MAX_ENTRIES / (WARPS * 32)) + x;
        if (i < a.n) {
            base[i] = scan + mine[x];
            if (blockIdx.x == 0) a.base[i] = scan + mine[x];
        }
    }
    if (tid == 0) {
        base[a.n] = total;
        if (blockIdx.x == 0) a.base[a.n] = total;
    }
    __syncthreads();
    // entries that see no tokens: rows of zeros
    for (uint32_t i = blockIdx.x; i < a.n; i += gridDim.x) {
        if (base[i + 1] != base[i]) continue;
        const Entry e = load_entry<NT>(a, i);
        const uint32_t width = a.H * DK;
        for (uint64_t x = tid; x < static_cast<uint64_t>(e.rows) * width; x += WARPS * 32)
            static_cast<T*>(a.o)[(e.r0 + x / width) * a.os + x % width] = c4_round<T>(0.0f);
    }
    // warps side by side in a share's order lie on different SMs
    const uint64_t w = static_cast<uint64_t>(warp) * gridDim.x + blockIdx.x;
    const uint64_t n_shares = shares(a, total, static_cast<uint64_t>(gridDim.x) * WARPS);
    if (w >= n_shares) return;
    const uint64_t begin = share_begin(w, total, n_shares), end = share_begin(w + 1, total, n_shares);
    uint8_t* ring = smem + warp * STAGES * BYTES;

    // where a tile lies: its entry, and its item within it
    auto entry_at = [&](uint64_t x) {
        uint32_t lo = 0, hi = a.n;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (base[mid] <= x) lo = mid; else hi = mid;
        }
        return lo;
    };
    // the producer's place: lanes 0 and 1 fetch a tile's two units
    uint64_t px = begin;
    Entry pe = {};
    uint32_t pi = 0, ptile = 0, ph = 0;
    uint64_t pitem = 0;
    auto p_enter = [&](uint64_t x) {
        pi = entry_at(x);
        pe = load_entry<NT>(a, pi);
        pitem = (x - base[pi]) / pe.tiles;
        ptile = static_cast<uint32_t>((x - base[pi]) % pe.tiles);
        ph = static_cast<uint32_t>(pitem / pe.blocks);
    };
    const uint8_t* src = nullptr;
    uint32_t fetch = 0;  // units of the next tile
    auto p_look = [&]() {
        if (px >= end) return;
        const uint32_t u = 2 * ptile;
        fetch = pe.units - u < 2 ? 1 : 2;
        src = nullptr;
        if (lane < fetch) {
            src = c4_unit(a.c, a.layer, pe.seq, ph, pe.unit0 + u + lane, a.err);
            // a table entry that is no page: any page will do, the rows are not defined
            if (!src) src = a.c.pages;
        }
    };
    auto p_issue = [&](int stage) {
        if (px >= end) return;
        if (lane == 0) mbar_arrive_expect_tx(&bars[warp][stage], fetch * 18 * DK);
        __syncwarp();
        if (lane < fetch) bulk_load(ring + stage * BYTES + lane * 18 * DK, src, 18 * DK, &bars[warp][stage]);
        px++;
        if (px < end) {
            if (++ptile == pe.tiles) {
                ptile = 0;
                if (++pitem == static_cast<uint64_t>(a.c.heads) * pe.blocks) p_enter(px);
                else ph = static_cast<uint32_t>(pitem / pe.blocks);
            }
            p_look();
        }
    };
    p_enter(px);
    p_look();
#pragma unroll
    for (int i = 0; i < STAGES; i++) p_issue(i);

    int stage = 0;
    uint32_t phase = 0;
    uint64_t x = begin;
    Entry e = {};
    uint32_t entry = FULL;
    while (x < end) {
        // one item, or the part of it in this share
        if (entry == FULL || x >= base[entry + 1]) {
            entry = entry_at(x);
            e = load_entry<NT>(a, entry);
        }
        const uint64_t item = (x - base[entry]) / e.tiles;
        const uint32_t first = static_cast<uint32_t>((x - base[entry]) % e.tiles);
        const uint32_t last = static_cast<uint32_t>(end - x < e.tiles - first ? first + (end - x) : e.tiles);
        const uint32_t h = static_cast<uint32_t>(item / e.blocks), block = static_cast<uint32_t>(item % e.blocks);
        Columns<NT> col;
        load_columns<NT>(a, e, h, block, col);
        uint32_t q[NB][2][NT][PARTS][2];
        {
            const uint32_t g = lane / 4, t = lane & 3;
            const uint64_t all = static_cast<uint64_t>(e.rows) * a.G;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const uint64_t r = static_cast<uint64_t>(block) * (8 * NT) + j * 8 + g;
                const T* qp = static_cast<const T*>(a.q) + (e.r0 + r / a.G) * a.qs + (static_cast<size_t>(h) * a.G + r % a.G) * DK + 8 * t;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float f[8];
#pragma unroll
                    for (int y = 0; y < 8; y++) f[y] = r < all ? c4_float<T>(qp[b * 32 + y]) : 0.0f;
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        uint32_t parts[PARTS];
                        bf16_parts<PARTS>(f[2 * y], f[2 * y + 1], parts);
#pragma unroll
                        for (int z = 0; z < PARTS; z++) q[b][y / 2][j][z][y % 2] = parts[z];
                    }
                }
            }
        }
        // the keys that every row of the block sees
        int32_t all_lo = 0, all_hi = INT_MAX;
#pragma unroll
        for (int i = 0; i < 2 * NT; i++)
            if (col.row[i] >= 0) {
                all_lo = max(all_lo, col.lo[i]);
                all_hi = min(all_hi, col.hi[i]);
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
        for (uint32_t tile = first; tile < last; tile++) {
            if (!mbar_wait(&bars[warp][stage], phase, &gave_up, a.timeout)) {
                // a copy that does not come: say so, let those in flight land, leave
                gave_up = 1;
                if (lane == 0) atomicOr(a.err, PKB_DEVERR_TIMEOUT);
                for (int i = 0; i < STAGES && x + i < px; i++) {
                    mbar_drain(&bars[warp][stage], phase, a.timeout);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
                return;
            }
            const uint8_t* buf = ring + stage * BYTES;
            const int32_t key0 = static_cast<int32_t>((e.unit0 + 2 * tile) * C4_UNIT);
            // warp-uniform: tiles at the window's start, the causal edge and the last token
            if (key0 < all_lo || static_cast<int64_t>(key0) + TILE > all_hi)
                tile_step<NB, NT, PARTS, true>(buf, q, col, key0, static_cast<int32_t>(e.len), a.scale, o, m, l);
            else
                tile_step<NB, NT, PARTS, false>(buf, q, col, key0, static_cast<int32_t>(e.len), a.scale, o, m, l);
            __syncwarp();
            p_issue(stage);
            x++;
            if (++stage == STAGES) stage = 0, phase ^= 1;
        }
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) l[i] = column_sum(l[i]);
        if (first == 0 && last == e.tiles) {
            write_rows<T, NB, NT>(a, col, o, l);
        } else {
            float* part = a.part + ((2 * w + (first == 0)) * part_regs<NB, NT>()) * 32 + lane;
#pragma unroll
            for (int d = 0; d < 2 * NB; d++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int y = 0; y < 4; y++) part[((d * NT + j) * 4 + y) * 32] = o[d][j][y];
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) {
                part[(NB * 8 * NT + i) * 32] = m[i];
                part[(NB * 8 * NT + 2 * NT + i) * 32] = l[i];
            }
        }
    }
}

// Joins the parts of the items that several shares have: one block an item,
// its warps take the parts in turn, then each other's, in the same order
// always.
template <typename T, int NB, int NT>
__global__ void __launch_bounds__(WARPS * 32) join_kernel(Attn4Args a, uint64_t warps) {
    constexpr int REGS = NB * 8 * NT;
    __shared__ float sm[WARPS][4 * NT][32];
    extern __shared__ float so[];  // [WARPS][REGS][32]
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t i = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads;
    const uint64_t total = a.base[a.n], first = a.base[i];
    if (a.base[i + 1] == first) return;
    const uint64_t n_shares = shares(a, total, warps);
    const Entry e = load_entry<NT>(a, i);
    for (uint32_t block = blockIdx.y; block < e.blocks; block += gridDim.y) {
        const uint64_t x0 = first + (static_cast<uint64_t>(h) * e.blocks + block) * e.tiles, x1 = x0 + e.tiles - 1;
        const uint64_t w0 = ((x0 + 1) * n_shares - 1) / total, w1 = ((x1 + 1) * n_shares - 1) / total;
        if (w0 == w1) continue;  // one share has it whole and wrote it
        float o[REGS], m[2 * NT], l[2 * NT];
#pragma unroll
        for (int r = 0; r < REGS; r++) o[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < 2 * NT; c++) m[c] = NEG_INF, l[c] = 0.0f;
        for (uint64_t w = w0 + warp; w <= w1; w += WARPS) {
            const float* part = a.part + ((2 * w + (w == w0)) * part_regs<NB, NT>()) * 32 + lane;
            float f[2 * NT], k[2 * NT];
#pragma unroll
            for (int c = 0; c < 2 * NT; c++) {
                const float pm = part[(REGS + c) * 32], pl = part[(REGS + 2 * NT + c) * 32];
                const float top = fmaxf(m[c], pm);
                k[c] = rescale(m[c], top);
                f[c] = rescale(pm, top);
                m[c] = top;
                l[c] = l[c] * k[c] + pl * f[c];
            }
#pragma unroll
            for (int r = 0; r < REGS; r++) {
                const int c = 2 * (r / 4 % NT) + r % 2;
                o[r] = o[r] * k[c] + part[r * 32] * f[c];
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2 * NT; c++) sm[warp][c][lane] = m[c], sm[warp][2 * NT + c][lane] = l[c];
#pragma unroll
        for (int r = 0; r < REGS; r++) so[(warp * REGS + r) * 32 + lane] = o[r];
        __syncthreads();
        // the rows' weights of each warp's sum, then REGS / WARPS of a row's values a warp
        float f[WARPS][2 * NT];
#pragma unroll
        for (int c = 0; c < 2 * NT; c++) {
            float top = NEG_INF;
#pragma unroll
            for (int w = 0; w < WARPS; w++) top = fmaxf(top, sm[w][c][lane]);
            l[c] = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                f[w][c] = rescale(sm[w][c][lane], top);
                l[c] += sm[w][2 * NT + c][lane] * f[w][c];
            }
        }
        Columns<NT> col;
        load_columns<NT>(a, e, h, block, col);
        const uint32_t g = lane / 4;
#pragma unroll
        for (int z = 0; z < REGS / WARPS; z++) {
            // registers of a lane: [dims 16][columns][row g, g + 8][two columns]
            const int r = z * WARPS + static_cast<int>(warp);
            float sum = 0.0f;
            const int j = r / 4 % NT, c = 2 * j + r % 2;
            float lc = 0.0f;
            int64_t row = -1;
            uint32_t head = 0;
#pragma unroll
            for (int y = 0; y < 2 * NT; y++)
                if (y == c) {
                    lc = l[y], row = col.row[y], head = col.head[y];
#pragma unroll
                    for (int w = 0; w < WARPS; w++) sum += so[(w * REGS + r) * 32 + lane] * f[w][y];
                }
            if (row < 0) continue;
            const float inv = lc == 0.0f ? 0.0f : __fdiv_rn(1.0f, lc);
            static_cast<T*>(a.o)[row * a.os + static_cast<size_t>(head) * (NB * 32) + r / (4 * NT) * 16 + r % 4 / 2 * 8 + g] =
                c4_round<T>(__fmul_rn(sum, inv));
        }
    }
}

// ------------------------------------------------------------------- host --

template <int NB> size_t split_smem(uint32_t n) { return WARPS * stages<NB>() * tile_bytes<NB>() + (static_cast<size_t>(n) + 1) * 8; }
template <int NB, int NT> size_t join_smem() { return static_cast<size_t>(WARPS) * NB * 8 * NT * 32 * 4; }

template <typename T, int NB, int NT, int PARTS>
cudaError_t prepare_one() {
    cudaError_t e = cudaFuncSetAttribute(split_kernel<T, NB, NT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(split_smem<NB>(MAX_ENTRIES)));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(join_kernel<T, NB, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(join_smem<NB, NT>()));
    return e;
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
cudaError_t launch_one(const Attn4Args& a, uint32_t max_rows, int sms, cudaStream_t s) {
    const uint32_t grid = static_cast<uint32_t>(blocks_per_sm<NB, NT, PARTS>() * sms < MAX_GRID ? blocks_per_sm<NB, NT, PARTS>() * sms : MAX_GRID);
    cudaError_t e = c4_launch(split_kernel<T, NB, NT, PARTS>, grid, WARPS * 32, split_smem<NB>(a.n), s, a);
    if (e != cudaSuccess) return e;
    count_launch();
    const uint64_t blocks = (static_cast<uint64_t>(max_rows) * a.G + 8 * NT - 1) / (8 * NT);
    const dim3 jgrid(a.n * a.c.heads, static_cast<uint32_t>(blocks < 1 ? 1 : blocks > 65535 ? 65535 : blocks));
    e = c4_launch(join_kernel<T, NB, NT>, jgrid, WARPS * 32, join_smem<NB, NT>(), s, a, static_cast<uint64_t>(grid) * WARPS);
    if (e == cudaSuccess) count_launch();
    return e;
}

template <typename T, int PARTS>
cudaError_t launch_type(const Attn4Args& a, uint32_t max_rows, int sms, cudaStream_t s) {
    const bool two = static_cast<uint64_t>(max_rows) * a.G > 8;  // more than eight rows: two blocks of eight share the codes' conversion
    switch (a.c.dk) {
        case 32: return two ? launch_one<T, 1, 2, PARTS>(a, max_rows, sms, s) : launch_one<T, 1, 1, PARTS>(a, max_rows, sms, s);
        case 64: return two ? launch_one<T, 2, 2, PARTS>(a, max_rows, sms, s) : launch_one<T, 2, 1, PARTS>(a, max_rows, sms, s);
        case 96: return two ? launch_one<T, 3, 2, PARTS>(a, max_rows, sms, s) : launch_one<T, 3, 1, PARTS>(a, max_rows, sms, s);
        case 128: return two ? launch_one<T, 4, 2, PARTS>(a, max_rows, sms, s) : launch_one<T, 4, 1, PARTS>(a, max_rows, sms, s);
        default: return launch_one<T, 8, 1, PARTS>(a, max_rows, sms, s);
    }
}

constexpr size_t BASE_BYTES = (MAX_ENTRIES + 32) * 8;

bool is_aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// The shares that a call can have at most, and the bytes of their parts.
uint64_t most_shares(const pkb_cache4* c, uint32_t H, uint32_t rows, uint32_t n) {
    const uint64_t tiles = static_cast<uint64_t>(c->max_pages) * c->page_tokens / TILE + 1;
    const uint64_t blocks = n + static_cast<uint64_t>(rows) * (H / c->n_heads) / 8;
    const uint64_t most = static_cast<uint64_t>(MAX_GRID) * WARPS;
    return blocks >= most || blocks * c->n_heads * tiles >= most ? most : blocks * c->n_heads * tiles;
}

size_t work_bytes_for(const pkb_cache4* c, uint32_t H, uint32_t rows, uint32_t n) {
    const uint64_t nt = c->head_dim == 256 ? 1 : 2;
    return BASE_BYTES + 2 * most_shares(c, H, rows, n) * nt * (c->head_dim / 4 + 4) * 128;
}

}  // namespace

cudaError_t prepare_attention4() {
    cudaError_t e = prepare_type<float, 3>();
    if (e == cudaSuccess) e = prepare_type<__half, 2>();
    if (e == cudaSuccess) e = prepare_type<__nv_bfloat16, 1>();
    return e;
}

}  // namespace pkb

using namespace pkb;

extern "C" {

size_t pkb_attention_cache4_work_bytes(const pkb_cache4* c, uint32_t H, uint32_t rows, uint32_t n) {
    if (!c || !pkb_cache4_page_bytes(c->page_tokens, c->n_heads, c->head_dim) || !H || H % c->n_heads) return 0;
    return work_bytes_for(c, H, rows, n);
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
    if (!(scale - scale == 0.0f)) return set_error(PKB_EINVAL, "%s: scale is not finite", who);
    if (window > INT_MAX) return set_error(PKB_EINVAL, "%s: window = %u", who, window);
    if (!n || !rows) return PKB_OK;
    if (!o || !q || !seqs || !starts || !work) return set_error(PKB_EINVAL, "%s: null pointer", who);
    if (!max_rows || max_rows > rows) return set_error(PKB_EINVAL, "%s: max_rows = %u of %u rows", who, max_rows, rows);
    const size_t width = static_cast<size_t>(H) * c->head_dim, size = c4_type_bytes(type);
    if (width > UINT_MAX / 2 || rows > INT_MAX) return set_error(PKB_EINVAL, "%s: %u rows of %zu values", who, rows, width);
    if (rows > 1 && (qs < width || os < width)) return set_error(PKB_EINVAL, "%s: a row stride below %zu values", who, width);
    if (rows == 1) qs = os = width;
    if (!is_aligned(o, size) || !is_aligned(q, size) || !is_aligned(seqs, 4) || !is_aligned(starts, 4))
        return set_error(PKB_EINVAL, "%s: misaligned buffer", who);
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), q1 = q0 + ((rows - 1) * qs + width) * size;
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(o), o1 = o0 + ((rows - 1) * os + width) * size;
    if (o0 < q1 && q0 < o1) return set_error(PKB_EINVAL, "%s: o overlaps q", who);
    const size_t need = work_bytes_for(c, H, rows, n);
    if (work_bytes < need || !is_aligned(work, 256))
        return set_error(PKB_EINVAL, "%s: work area of %zu bytes (%zu needed, 256-byte aligned)", who, work_bytes, need);
    if (static_cast<uint64_t>(MAX_ENTRIES) * c->n_heads > INT_MAX) return set_error(PKB_EINVAL, "%s: %u heads", who, c->n_heads);
    int sms;
    if ((rc = current_device_info(&sms, &a.err))) return rc;
    a.q = q;
    a.o = o;
    a.qs = qs;
    a.os = os;
    a.layer = layer;
    a.rows = rows;
    a.H = H;
    a.G = H / c->n_heads;
    a.scale = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634074);  // log2 e
    a.causal = causal ? 1 : 0;
    a.window = window;
    a.timeout = wait_cycles();
    a.base = static_cast<uint64_t*>(work);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + BASE_BYTES);
    a.max_shares = most_shares(c, H, rows, n);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    for (uint32_t i = 0; i < n; i += MAX_ENTRIES) {
        a.seqs = seqs + i;
        a.starts = starts + i;
        a.n = n - i < MAX_ENTRIES ? n - i : MAX_ENTRIES;
        const cudaError_t e = type == PKB_F32   ? launch_type<float, 3>(a, max_rows, sms, s)
                              : type == PKB_F16 ? launch_type<__half, 2>(a, max_rows, sms, s)
                                                : launch_type<__nv_bfloat16, 1>(a, max_rows, sms, s);
        if (e != cudaSuccess)
            return set_error(e == cudaErrorMemoryAllocation ? PKB_ENOMEM : PKB_ECUDA, "%s launch: %s", who, cudaGetErrorString(e));
    }
    return PKB_OK;
}

}  // extern "C"
