// The cache held in 4 bits, as kernels see it: where a unit lies, and the
// codes' way to and from bf16 (include/pktito_b200.h, pkb_cache4).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pktito_b200.h"

namespace pkb {

constexpr int C4_UNIT = 16;   // tokens of a unit
constexpr int C4_BLOCK = 32;  // values of a scale

// pkb_cache4 with what its sizes give, one layer's pages
struct Cache4 {
    uint8_t* pages;
    int32_t *table, *lens, *refs;
    uint32_t n_layers, n_pages, max_seqs, max_pages, heads, dk;
    uint32_t pshift;         // page_tokens = 1 << pshift
    uint32_t unit_bytes;     // 18 dk
    size_t head_bytes;       // a head's units of one page
    size_t page_bytes, layer_bytes;
};

// Token `unit`'s sixteen of head h: the unit's bytes (*users: how many
// sequences hold its page), or null (*err set) where the table names no page.
__device__ __forceinline__ uint8_t* c4_unit(const Cache4& c, uint32_t layer, uint32_t seq, uint32_t h, uint32_t unit,
                                            const int32_t** users, uint32_t* err) {
    const uint32_t per = c.pshift - 4;  // log2 of the units of a page
    const int32_t page = c.table[static_cast<size_t>(seq) * c.max_pages + (unit >> per)];
    if (page < 0 || static_cast<uint32_t>(page) >= c.n_pages) {
        atomicOr(err, 2u);
        return nullptr;
    }
    *users = c.refs + page;
    return c.pages + layer * c.layer_bytes + static_cast<size_t>(page) * c.page_bytes + h * c.head_bytes +
           (unit & ((1u << per) - 1)) * static_cast<size_t>(c.unit_bytes);
}

// A sequence's tokens, within what its table row has room for.
__device__ __forceinline__ uint32_t c4_len(const Cache4& c, uint32_t seq, uint32_t* err) {
    const int32_t len = c.lens[seq];
    if (len < 0 || static_cast<uint64_t>(len) > static_cast<uint64_t>(c.max_pages) << c.pshift) {
        atomicOr(err, 2u);
        return 0;
    }
    return static_cast<uint32_t>(len);
}

// Rows [*r0, *r0 + count) of entry i of a call; 0 where starts or the
// sequence are out of range (*err set, unless the entry has no rows: a
// padded batch may name no sequence there).
__device__ __forceinline__ uint32_t c4_rows(const Cache4& c, const int32_t* seqs, const int32_t* starts, uint32_t i,
                                            uint32_t rows, uint32_t* seq, uint32_t* r0, uint32_t* err) {
    const int32_t a = starts[i], b = starts[i + 1], s = seqs[i];
    *r0 = static_cast<uint32_t>(a);
    *seq = static_cast<uint32_t>(s);
    if (a < 0 || b < a || static_cast<uint32_t>(b) > rows || s < 0 || static_cast<uint32_t>(s) >= c.max_seqs) {
        if (a != b) atomicOr(err, 2u);
        *seq = 0;
        return 0;
    }
    return static_cast<uint32_t>(b - a);
}

// The four pairs of a word's eight codes as bf16 pairs, each a quarter of
// what it stands for: a nibble n in the top four mantissa bits of 4.0 is
// (16 + n) / 4, and the one fused (16 + n) / 4 s - 6 s is c s / 4 exactly (6 s
// has 7 significant bits, c s 8), so neither the conversion nor the scale
// rounds. Three instructions a pair. The quarter keeps 6 s finite for every
// scale (24 s is not from 2^123 on, and a masked weight's 0 times it is a NaN in rows that do
// not see the key), and c s / 4 normal for the smallest.
template <int J, uint32_t BASE>
__device__ __forceinline__ uint32_t c4_placed(uint32_t w) {
    const uint32_t at = J == 0 ? w << 3 : w >> (4 * J - 3);
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(r) : "r"(at), "n"(BASE));  // (at & mask) | BASE
    return r;
}
template <int J>
__device__ __forceinline__ uint32_t c4_quarter(uint32_t w, uint32_t s2, uint32_t m6s2) {
    uint32_t r = c4_placed<J, 0x40804080u>(w);  // 4.0
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(r), "r"(s2), "r"(m6s2));
    return r;
}

// The whole of it, in four instructions: 16 + n less 24 first.
template <int J>
__device__ __forceinline__ uint32_t c4_whole_pair(uint32_t w, uint32_t s2) {
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(c4_placed<J, 0x41804180u>(w)), "r"(0xC1C0C1C0u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(s2));
    return r;
}

// -6 s of both halves
__device__ __forceinline__ uint32_t c4_m6(uint32_t s2) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(s2), "r"(0xC0C0C0C0u));
    return r;
}

// a bf16's bits as a float
__device__ __forceinline__ float c4_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }

template <typename T> __device__ __forceinline__ float c4_float(T v);
template <> __device__ __forceinline__ float c4_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float c4_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float c4_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T c4_round(float v);
template <> __device__ __forceinline__ float c4_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half c4_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 c4_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight values at p, sixteen bytes at a time where VEC (p 16-byte aligned).
template <typename T, bool VEC>
__device__ __forceinline__ void c4_load8(const T* p, float (&x)[8]) {
    alignas(16) T v[8];
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; i++)
            reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = c4_float<T>(v[i]);
}

template <typename T, bool VEC>
__device__ __forceinline__ void c4_store8(T* p, const float (&x)[8]) {
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = c4_round<T>(x[i]);
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; i++)
            reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = v[i];
    }
}

// host: checks the descriptor and gives the kernels' view (pkb_cache4.cu)
int c4_view(const pkb_cache4* c, const char* who, Cache4* out);
int c4_check_type(int type, const char* who);
inline size_t c4_type_bytes(int type) { return type == PKB_F32 ? 4 : 2; }

// host: one launch on the stream, allowed to begin while the kernel before
// it ends (each kernel waits for that one's results by pdl_wait)
template <typename... P, typename... A>
inline cudaError_t c4_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace pkb
