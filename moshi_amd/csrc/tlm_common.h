// What the token language models' kernels and operators share: operand formats, fragment-packed matrices, masks, pages.
#pragma once
#include "mmi_common.h"

struct TlmBf16 {
    typedef uint16_t elem;
    static constexpr int V = 8, KSTEP = 32;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) { return mmi_mfma_bf16_16x16x32(a, b, c); }
    static __device__ __forceinline__ uint16_t cvt(float v) { return mmi_f32_to_bf16(v); }
    static __device__ __forceinline__ void store4(uint16_t* p, f32x4 v) {
        u32x2 o = {mmi_pack_bf16x2(v[0], v[1]), mmi_pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2*>(p) = o;
    }
    static __device__ __forceinline__ void store2(uint16_t* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = mmi_pack_bf16x2(a, b); }
};
struct TlmF32 {
    typedef float elem;
    static constexpr int V = 4, KSTEP = 16;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = mmi_mfma_f32_16x16x4(fa[e], fb[e], c);
        return c;
    }
    static __device__ __forceinline__ float cvt(float v) { return v; }
    static __device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
    static __device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<f32x2*>(p) = f32x2{a, b}; }
};

// element (row, k) of a fragment-packed matrix with `ks` k-steps per row tile
template <class Tr>
MMI_HD long tlm_index(long row, int k, int ks) {
    return (((row >> 4) * ks + k / Tr::KSTEP) * 64 + ((k % Tr::KSTEP) / Tr::V) * 16 + (row & 15)) * Tr::V + k % Tr::V;
}

constexpr int TLM_PAGE = 64;         // tokens per cache page

// which keys a position sees, and the factor of the scores (times log2(e)): the last `window` ones (0: all), and the first `keep`
struct TlmMask { int window, keep; float scale; };
constexpr int TLM_KEEP = 0x7fffff00;      // more first positions than there can be; rounded up to pages it has 31 bits still
// pages of a sequence: the block table's first `keep` entries are for the pages that no window releases, the others are a ring
struct TlmPages { const int* table; int ld, keep; };
__device__ __forceinline__ int tlm_page(const TlmPages& p, const int* row, int i) { return mmi_load_const(row + (i < p.keep ? i : p.keep + (i - p.keep) % (p.ld - p.keep))); }
