// A paged key/value cache in 8 bits, and the attention over it.
//
//   page         64 tokens of every key/value head; block: 16 tokens of it, with one scale per head for the keys and one for the values
//   key codes    [page][head][64][dim]           value codes  [page][head][vdim][64]          scales  [page][head][4], fp32
//   value        code * scale of its block; int8: codes -127 .. 127, e4m3: -448 .. 448
//
// A block's scale is max(the scale it has, the largest magnitude it is handed / the largest code): where tokens make it grow, the codes the
// block holds already are rounded again.  A NaN or an infinity makes the block's scale NaN, and with it everything that attends to the block.
//
// Both layouts are what the matrix core takes, by wide loads without a turn through LDS: a lane (l & 15, kq = l >> 4) brings 16 bytes of one
// key - 16 dimensions, two k-steps of 8 - or 16 bytes of one value dimension - the 16 tokens of block kq.  For the weights of those 16 tokens
// to be in that lane when the scores are done, row 4 a + i of score tile t is token 16 a + 4 t + i: lane kq then holds, over the four tiles,
// the scores of block kq's tokens in order, and one key scale and one value scale are all it needs.
// Codes become bf16 exactly (8 bits at most), so fp32 queries and weights go through the bf16 matrix core in three parts of 8 bits each.
#pragma once
#include "tlm_common.h"

constexpr int KV8_BLOCK = 16, KV8_PARTS = TLM_PAGE / KV8_BLOCK;
constexpr float KV8_TINY = 7.8886090522101181e-31f;        // 2^-100: smallest magnitude that a block's scale is made from

struct TlmKv8Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    int n_pages, kv_heads, dim, vdim, e4m3;
    int rot, halves;                     // dimensions that are rotated; partners half of them apart, or side by side
    const double* freq;                  // [rot / 2] turns per position
};

// the sequences of a call: rows row0[e] .. of the call's tensors are positions pos0[e] .. of entry e
struct TlmKv8Seqs {
    int n, T;
    const int* row0;                     // null: one row each
    const int* len;                      // null: up to row0[e + 1]
    const int* pos0;
    const int* slot;                     // block table row of an entry; null: its own
    TlmPages pages;
    int ring;                            // the block table's entries past `keep` are a ring (tlm_page); otherwise entry i is page i, and there are `ld`
};

struct TlmKv8Seq { int e, row0, len, pos0; };
__device__ __forceinline__ int kv8_row0(const TlmKv8Seqs& a, int e) { return a.row0 ? min(max(a.row0[e], 0), a.T) : min(e, a.T); }
// (whatever the device arrays hold, rows stay inside the call's tensors and positions inside 31 bits)
__device__ __forceinline__ TlmKv8Seq kv8_seq(const TlmKv8Seqs& a, int e) {
    TlmKv8Seq s;
    s.e = e;
    s.row0 = mmi_uniform(kv8_row0(a, e));
    const int len = a.len ? a.len[e] : (a.row0 ? a.row0[e + 1] - a.row0[e] : 1), pos0 = a.pos0[e];
    s.len = mmi_uniform(pos0 < 0 || pos0 > 0x7fffff00 - a.T ? 0 : min(max(len, 0), a.T - s.row0));
    s.pos0 = mmi_uniform(pos0);
    return s;
}
// page number of the sequence's tokens 64 i .. 64 i + 63; -1: there is none
__device__ __forceinline__ int kv8_page(const TlmKv8Seqs& a, int n_pages, const int* row, int i) {
    if (!a.ring && i >= a.pages.ld) return -1;
    const int p = a.ring ? tlm_page(a.pages, row, i) : mmi_load_const(row + i);
    return p < 0 || p >= n_pages ? -1 : p;
}
__device__ __forceinline__ const int* kv8_table(const TlmKv8Seqs& a, int e) { return a.pages.table + (long)mmi_uniform(a.slot ? a.slot[e] : e) * a.pages.ld; }

// An entry's work is cut into pieces of `per` units, `mul` units a row, without anyone having counted them: entry e owns the slots from
// row0[e] * mul / per + extra e on, which are as many as it can need, and a slot's entry is the last one that begins at or before it.
// One row each: `extra` slots per entry.
struct Kv8Cut { int mul, per, extra; };
__device__ __forceinline__ int kv8_slot0(const TlmKv8Seqs& a, const Kv8Cut& z, int e) { return (a.row0 ? (int)((long)kv8_row0(a, e) * z.mul / z.per) : 0) + z.extra * e; }
__device__ __forceinline__ int kv8_find(const TlmKv8Seqs& a, const Kv8Cut& z, int slot) {
    if (!a.row0) return min(slot / z.extra, a.n - 1);
    unsigned below = 0;
    for (int e = mmi_lane(); e < a.n; e += 64) below += kv8_slot0(a, z, e) <= slot ? 1u : 0u;
    return max(mmi_uniform((int)mmi_wave_sum_u32(below) - 1), 0);
}
// host: the cut of `units` = mul * rows units, and how many slots there are
inline Kv8Cut kv8_cut(const TlmKv8Seqs& a, int mul, int per, int more) { return Kv8Cut{mul, per, a.row0 ? more : mmi_cdiv(mul, per)}; }
inline long kv8_slots(const TlmKv8Seqs& a, const Kv8Cut& z) { return (a.row0 ? (long)a.T * z.mul / z.per : 0) + (long)z.extra * a.n; }

// ---- codes ---------------------------------------------------------------------------------------------------------------
template <bool E4M3>
struct Kv8Code {
    static constexpr float TOP = E4M3 ? 448.f : 127.f;
    static __device__ __forceinline__ uint32_t pack(f32x4 x) {
        if constexpr (E4M3) return mmi_cvt_fp8x4(x[0], x[1], x[2], x[3]);
        int c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = (int)mmi_rint(fminf(fmaxf(x[i], -127.f), 127.f));
        return mmi_pack_low_bytes((uint32_t)c[0], (uint32_t)c[1], (uint32_t)c[2], (uint32_t)c[3]);
    }
    static __device__ __forceinline__ f32x4 unpack(uint32_t w) {
        f32x4 o;
        if constexpr (E4M3) {
            float f[4];
            mmi_fp8x4_to_f32(w, f);
            o = f32x4{f[0], f[1], f[2], f[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = (float)((int)(w << (24 - 8 * i)) >> 24);
        }
        return o;
    }
    static __device__ __forceinline__ u32x2 bf16(uint32_t w) {
        if constexpr (E4M3) return mmi_fp8x4_to_bf16(w);
        const f32x4 f = unpack(w);
        return u32x2{mmi_pack_bf16x2(f[0], f[1]), mmi_pack_bf16x2(f[2], f[3])};
    }
    // 16 codes -> two operand fragments of 8
    static __device__ __forceinline__ void fragments(u32x4 c, u32x4& lo, u32x4& hi) {
        const u32x2 a = bf16(c[0]), b = bf16(c[1]), d = bf16(c[2]), e = bf16(c[3]);
        lo = u32x4{a[0], a[1], b[0], b[1]};
        hi = u32x4{d[0], d[1], e[0], e[1]};
    }
};

__device__ __forceinline__ float kv8_load(const float* p) { return *p; }
__device__ __forceinline__ float kv8_load(const uint16_t* p) { return mmi_bf16_to_f32(*p); }
__device__ __forceinline__ f32x4 kv8_load4(const float* p) { return *(const f32x4*)p; }
__device__ __forceinline__ f32x4 kv8_load4(const uint16_t* p) {
    const u32x2 w = *(const u32x2*)p;
    return f32x4{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16),
                 __builtin_bit_cast(float, w[1] & 0xffff0000u)};
}
template <class In>
__device__ __forceinline__ f32x4 kv8_in4(const In* p, bool wide) {
    if (wide) return kv8_load4(p);
    return f32x4{kv8_load(p), kv8_load(p + 1), kv8_load(p + 2), kv8_load(p + 3)};
}
// the angle's turns are formed in 64 bits and reduced there: at position 2^20 a turn's fraction would have 3 bits left in fp32
__device__ __forceinline__ void kv8_angle(int pos, double freq, float& c, float& s) {
    const double t = (double)pos * freq;
    mmi_sincos_turns((float)(t - rint(t)), s, c);
}
// dimensions d .. d + 3 (d a multiple of 4) of a row, rotated
template <class In>
__device__ __forceinline__ f32x4 kv8_rotated4(const In* row, int d, int pos, int rot, int halves, const double* freq, bool wide) {
    f32x4 x = kv8_in4(row + d, wide);
    if (d >= rot) return x;
    if (halves) {
        const int h = rot / 2, i = d < h ? d : d - h;
        const f32x4 y = kv8_in4(row + (d < h ? d + h : d - h), wide);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float c, s, re, im;
            kv8_angle(pos, freq[i + r], c, s);
            mmi_rope_rotate(d < h ? x[r] : y[r], d < h ? y[r] : x[r], c, s, re, im);
            x[r] = d < h ? re : im;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            float c, s, re, im;
            kv8_angle(pos, freq[(d + r) / 2], c, s);
            mmi_rope_rotate(x[r], x[r + 1], c, s, re, im);
            x[r] = re;
            x[r + 1] = im;
        }
    }
    return x;
}

// ---- append --------------------------------------------------------------------------------------------------------------
struct TlmKv8Append {
    TlmKv8Cache c;
    TlmKv8Seqs q;
    Kv8Cut z;                            // of rows, by blocks
    const void *k, *v;
    long k_row, k_head, v_row, v_head;   // strides in elements; a head's dimensions lie side by side
    int wide;                            // every 4 elements are aligned
};

// a block of an entry: tokens lo .. hi - 1 of its 16 are new, the ones before are held already
struct Kv8Span { int page, part, lo, hi, row, pos; bool none; };
__device__ __forceinline__ Kv8Span kv8_span(const TlmKv8Seqs& q, const Kv8Cut& z, int n_pages, int slot) {
    const int e = kv8_find(q, z, slot);
    const TlmKv8Seq s = kv8_seq(q, e);
    const int b = s.pos0 / KV8_BLOCK + slot - kv8_slot0(q, z, e);      // block of the sequence
    Kv8Span o;
    o.pos = b * KV8_BLOCK;
    o.none = s.len < 1 || o.pos >= s.pos0 + s.len;
    o.lo = max(s.pos0 - o.pos, 0);
    o.hi = min(s.pos0 + s.len - o.pos, KV8_BLOCK);
    o.row = s.row0 + o.pos - s.pos0;               // row of the block's first token (of token lo on they are the call's)
    o.page = o.none ? -1 : kv8_page(q, n_pages, kv8_table(q, e), b / KV8_PARTS);
    o.part = b % KV8_PARTS;
    o.none = o.none || o.page < 0;
    return o;
}
// scale of the block after tokens with the largest magnitude `bits` (as an integer: a NaN's is above all others)
template <bool E4M3>
__device__ __forceinline__ float kv8_grown(float before, bool held, unsigned bits, float& ratio) {
    const float top = fmaxf(__builtin_bit_cast(float, bits), KV8_TINY) / Kv8Code<E4M3>::TOP;
    float after = fmaxf(before, top);
    if (bits >= 0x7f800000u || !(before < INFINITY)) after = __builtin_bit_cast(float, 0x7fc00000u);
    ratio = held ? before / after : 1.f;
    return after;
}
__device__ __forceinline__ unsigned kv8_bits(f32x4 x) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = x[i];                              // (a bit cast of a vector's element itself takes element 0)
        m = max(m, __builtin_bit_cast(unsigned, y) & 0x7fffffffu);
    }
    return m;
}

// One wave per block, head and side.  grid: slots of blocks, kv heads, 2 (keys, values)
//   keys: four lanes per token, granules of 4 dimensions in turn      values: a lane per dimension, its 16 tokens side by side
template <class In, bool E4M3>
__global__ __launch_bounds__(64) void k_tlm_kv8_append(TlmKv8Append a) {
    typedef Kv8Code<E4M3> C;
    const Kv8Span s = kv8_span(a.q, a.z, a.c.n_pages, (int)blockIdx.x);
    if (s.none) return;
    const int lane = mmi_lane(), g = (int)blockIdx.y, part = s.part;
    const bool held = s.lo > 0, wide = a.wide != 0;
    const long unit = (long)s.page * a.c.kv_heads + g;
    if (blockIdx.z == 0) {
        const int t = lane >> 2, c = lane & 3, n = a.c.dim / 16;
        const In* row = (const In*)a.k + (long)(s.row + t) * a.k_row + g * a.k_head;
        uint32_t* out = (uint32_t*)(a.c.k + (unit * TLM_PAGE + part * KV8_BLOCK + t) * a.c.dim);
        const bool fresh = t >= s.lo && t < s.hi;
        f32x4 x[16];
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n && fresh) {
                x[i] = kv8_rotated4(row, 4 * (c + 4 * i), s.pos + t, a.c.rot, a.c.halves, a.c.freq, wide);
                bits = max(bits, kv8_bits(x[i]));
            }
        float* scale = a.c.ks + unit * KV8_PARTS + part, ratio;
        const float before = held ? *scale : 0.f;
        bits = mmi_wave_max_u32(bits);
        const float after = kv8_grown<E4M3>(before, held, bits, ratio), inv = 1.f / after;
        const bool bad = !(after == after);
        if (fresh) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n) out[c + 4 * i] = bad ? 0u : C::pack(x[i] * inv);
        } else if (t < s.lo && ratio != 1.f) {
            for (int i = 0; i < n; ++i) out[c + 4 * i] = bad ? 0u : C::pack(C::unpack(out[c + 4 * i]) * ratio);
        }
        if (lane == 0) *scale = after;
    } else {
        const int n = (a.c.vdim + 63) / 64;
        const In* v = (const In*)a.v + (long)s.row * a.v_row + g * a.v_head;
        float x[4][KV8_BLOCK];
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d < a.c.vdim)
#pragma unroll
                for (int t = 0; t < KV8_BLOCK; ++t)
                    if (t >= s.lo && t < s.hi) {
                        x[i][t] = kv8_load(v + (long)t * a.v_row + d);
                        bits = max(bits, __builtin_bit_cast(unsigned, x[i][t]) & 0x7fffffffu);
                    }
        }
        float* scale = a.c.vs + unit * KV8_PARTS + part, ratio;
        const float before = held ? *scale : 0.f;
        bits = mmi_wave_max_u32(bits);
        const float after = kv8_grown<E4M3>(before, held, bits, ratio), inv = 1.f / after;
        const bool bad = !(after == after), whole = s.lo == 0 && s.hi == KV8_BLOCK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (i >= n || d >= a.c.vdim) continue;
            u32x4* out = (u32x4*)(a.c.v + (unit * a.c.vdim + d) * TLM_PAGE + part * KV8_BLOCK);
            u32x4 w = whole ? u32x4{0u, 0u, 0u, 0u} : *out;      // (the bytes behind the last token stay what they are)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 4 * j + r;
                    y[r] = t >= s.lo && t < s.hi ? x[i][t] * inv : 0.f;
                }
                const uint32_t now = bad ? 0u : C::pack(y), was = bad ? 0u : (ratio != 1.f ? C::pack(C::unpack(w[j]) * ratio) : w[j]);
                uint32_t m = 0, o = 0;                       // bytes of the new tokens, of the ones held
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 4 * j + r;
                    m |= t >= s.lo && t < s.hi ? 0xffu << (8 * r) : 0u;
                    o |= t < s.lo ? 0xffu << (8 * r) : 0u;
                }
                w[j] = (now & m) | (was & o) | (w[j] & ~(m | o));
            }
            *out = w;
        }
        if (lane == 0) *scale = after;
    }
}

// ---- read: the values that the cache holds for the call's rows --------------------------------------------------------------
struct TlmKv8Read {
    TlmKv8Cache c;
    TlmKv8Seqs q;
    Kv8Cut z;
    void *k, *v;                         // [rows][kv heads][dim], [rows][kv heads][vdim]; tokens without a page: zeros
};
__device__ __forceinline__ void kv8_put4(float* p, f32x4 v) { TlmF32::store4(p, v); }
__device__ __forceinline__ void kv8_put4(uint16_t* p, f32x4 v) { TlmBf16::store4(p, v); }
__device__ __forceinline__ void kv8_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void kv8_put(uint16_t* p, float v) { *p = mmi_f32_to_bf16(v); }
// grid: slots of blocks, kv heads, 2
template <class Out, bool E4M3>
__global__ __launch_bounds__(64) void k_tlm_kv8_read(TlmKv8Read a) {
    typedef Kv8Code<E4M3> C;
    Kv8Span s = kv8_span(a.q, a.z, a.c.n_pages, (int)blockIdx.x);
    if (s.none && s.hi <= s.lo) return;
    const int lane = mmi_lane(), g = (int)blockIdx.y;
    const long unit = (long)max(s.page, 0) * a.c.kv_heads + g;
    const float scale = s.none ? 0.f : (blockIdx.z ? a.c.vs : a.c.ks)[unit * KV8_PARTS + s.part];
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (blockIdx.z == 0) {
        const int t = lane >> 2, c = lane & 3;
        if (t < s.lo || t >= s.hi) return;
        const uint32_t* in = (const uint32_t*)(a.c.k + (unit * TLM_PAGE + s.part * KV8_BLOCK + t) * a.c.dim);
        Out* out = (Out*)a.k + ((long)(s.row + t) * a.c.kv_heads + g) * a.c.dim;
        for (int i = c; i < a.c.dim / 4; i += 4) kv8_put4(out + 4 * i, s.none ? zero : C::unpack(in[i]) * scale);
    } else {
        for (int d = lane; d < a.c.vdim; d += 64) {
            const u32x4 w = *(const u32x4*)(a.c.v + (unit * a.c.vdim + d) * TLM_PAGE + s.part * KV8_BLOCK);
            Out* out = (Out*)a.v + ((long)s.row * a.c.kv_heads + g) * a.c.vdim + d;
            const long ld = (long)a.c.kv_heads * a.c.vdim;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 x = s.none ? zero : C::unpack(w[j]) * scale;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (4 * j + r >= s.lo && 4 * j + r < s.hi) kv8_put(out + (4 * j + r) * ld, x[r]);
            }
        }
    }
}

// ---- attention -----------------------------------------------------------------------------------------------------------
struct TlmKv8Attn {
    TlmKv8Cache c;
    TlmKv8Seqs q;
    Kv8Cut z;                            // of columns (token, head of the group), by tiles
    const void* x; long x_row, x_head;   // queries
    int wide;                            // every 4 of their elements are aligned
    void* out; long out_row, out_head;   // rows; out_ks > 0: fragment-packed rows (tlm_index), columns head * 16 nd + d
    int out_ks;
    int heads, rep, nd;                  // rep: query heads per key/value head; nd: vdim / 16
    TlmMask mask;                        // scale: log2 e times the softmax's
    int sink;                            // one is added to the denominator
    int per, nsplit;                     // pages per split; splits that a tile can need
    float* po;                           // nsplit > 1: [tile slot][kv head][split][16 columns][vdim] un-normalised sums
    float* pml;                          // [tile slot][kv head][split][2][16]: running maximum, sum of weights
};

// columns (token, head of the group) c0 .. c0 + 15 of one entry, and the pages that they see: [0, n0) and [b0, b1)
struct Kv8Cols {
    TlmKv8Seq s;
    int c0, ncol, plo, phi, n0, b0, n;
    __device__ __forceinline__ Kv8Cols(const TlmKv8Attn& a, int slot) {
        const int e = kv8_find(a.q, a.z, slot), per = a.z.per;
        s = kv8_seq(a.q, e);
        c0 = (slot - kv8_slot0(a.q, a.z, e)) * per;
        ncol = s.len * a.rep;
        if (c0 >= ncol) {
            n = n0 = b0 = 0;
            return;
        }
        plo = s.pos0 + c0 / a.rep;
        phi = s.pos0 + min(c0 + per - 1, ncol - 1) / a.rep;
        const int w = a.mask.window;
        b0 = w > 0 && plo - w + 1 > 0 ? (plo - w + 1) / TLM_PAGE : 0;
        n0 = w > 0 ? min(b0, (a.mask.keep + TLM_PAGE - 1) / TLM_PAGE) : 0;
        n = n0 + phi / TLM_PAGE + 1 - b0;
        if (!a.q.ring) n = min(n, n0 + max(a.q.pages.ld - b0, 0));
    }
    __device__ __forceinline__ int page(int i) const { return i < n0 ? i : b0 + i - n0; }
    __device__ __forceinline__ bool seen(const TlmMask& m, int pos, int key) const { return key <= pos && (m.window <= 0 || pos - key < m.window || key < m.keep); }
    // every column sees the whole page
    __device__ __forceinline__ bool whole(const TlmMask& m, int key0) const { return key0 + TLM_PAGE - 1 <= plo && (m.window <= 0 || phi - key0 < m.window || key0 + TLM_PAGE <= m.keep); }
};

// fp32 -> NS parts of 8 bits of significand, pairs packed
template <int NS>
__device__ __forceinline__ void kv8_split2(float a, float b, uint32_t (&o)[NS]) {
#pragma unroll
    for (int p = 0; p < NS; ++p) {
        o[p] = mmi_pack_bf16x2(a, b);
        if (p + 1 < NS) {
            a -= __builtin_bit_cast(float, o[p] << 16);
            b -= __builtin_bit_cast(float, o[p] & 0xffff0000u);
        }
    }
}

// e4m3 bytes of tokens that no column sees may hold anything, a NaN among it, which a weight of zero would not silence: cleared
template <bool E4M3>
__device__ __forceinline__ u32x4 kv8_quiet(const Kv8Cols& c, const TlmMask& m, int key0, u32x4 w) {
    if constexpr (!E4M3) return w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t keep = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = key0 + 4 * j + r;
            keep |= key <= c.phi && (m.window <= 0 || c.plo - key < m.window || key < m.keep) ? 0xffu << (8 * r) : 0u;
        }
        w[j] &= keep;
    }
    return w;
}

// four dimensions of a row's head
template <class Tr>
__device__ __forceinline__ void kv8_store(const TlmKv8Attn& a, int row, int head, int d, f32x4 v) {
    typedef typename Tr::elem E;
    Tr::store4((E*)a.out + (a.out_ks ? tlm_index<Tr>(row, head * 16 * a.nd + d, a.out_ks) : row * a.out_row + head * a.out_head + d), v);
}

// Four waves share one tile of 16 columns, each takes every fourth of its pages and their sums meet in LDS.
// LDS: angles of the tile's tokens, then (the same memory) the waves' sums
constexpr int KV8_LDS = 4 * 8 * 64;                        // vectors of four floats
template <class In, class Tr, int NS, int D, bool E4M3>
__device__ __forceinline__ void tlm_kv8_attn(const TlmKv8Attn& a, f32x4* ob, float (*ml)[4][16], int slot, int g, int split) {
    typedef Kv8Code<E4M3> C;
    constexpr int NP = D / 64, ND = D / 16, WK = 4;
    const int lane = (int)threadIdx.x & 63, wave = mmi_uniform((int)threadIdx.x >> 6), bl = lane & 15, kq = lane >> 4;
    const Kv8Cols c(a, slot);
    const int i0 = split * a.per, i1 = min(c.n, i0 + a.per);
    if (c.c0 >= c.ncol || (i0 >= i1 && split > 0)) return;
    const int col = min(c.c0 + bl, c.ncol - 1), tok = col / a.rep, pos = c.s.pos0 + tok;
    const int* bt = kv8_table(a.q, c.s.e);
    u32x4 kf[4][NP], vf[ND];
    float ks = 0.f, vs = 0.f;
    int nb = 0;
    bool have = false;
    // (past the end, and where there is no page: the pool's first one, unused)
    auto load = [&](int i) __attribute__((always_inline)) {
        nb = c.page(min(i, i1 - 1));
        const int p = kv8_page(a.q, a.c.n_pages, bt, nb);
        have = p >= 0;
        const long unit = (long)max(p, 0) * a.c.kv_heads + g;
        const uint8_t* kp = a.c.k + (unit * TLM_PAGE + 16 * (bl >> 2) + (bl & 3)) * a.c.dim + 16 * kq;
        const uint8_t* vp = a.c.v + (unit * a.c.vdim + bl) * TLM_PAGE + 16 * kq;
        ks = a.c.ks[unit * KV8_PARTS + kq];
        vs = a.c.vs[unit * KV8_PARTS + kq];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) kf[t][p] = mmi_load_nt((const u32x4*)(kp + 4 * t * a.c.dim + (64 * p + 16 * kq < a.c.dim ? 64 * p : 0)));
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[d] = mmi_load_nt((const u32x4*)(vp + min(d, a.nd - 1) * 16 * TLM_PAGE));
    };
    if (i0 + wave < i1) load(i0 + wave);
    // the columns' queries, rotated: the tile's tokens are few, so their angles are formed once
    float* angle = reinterpret_cast<float*>(ob);           // [token of the tile][rot / 2][cos, sin]
    const int t0 = c.c0 / a.rep, nt = min(c.c0 + 15, c.ncol - 1) / a.rep - t0 + 1, half = a.c.rot / 2;
    for (int i = (int)threadIdx.x; i < nt * half; i += 256) kv8_angle(c.s.pos0 + t0 + i / half, a.c.freq[i % half], angle[2 * i], angle[2 * i + 1]);
    __syncthreads();
    u32x4 q[NS][2 * NP];
    {
        const In* row = (const In*)a.x + (long)(c.s.row0 + tok) * a.x_row + (g * a.rep + col - tok * a.rep) * a.x_head;
        const float* an = angle + (tok - t0) * 2 * half;
#pragma unroll
        for (int p = 0; p < 2 * NP; ++p) {                 // dimensions 64 (p / 2) + 16 kq + 8 (p & 1) ..
            const int d0 = 64 * (p >> 1) + 16 * kq + 8 * (p & 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = d0 + 4 * h;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (d < a.c.dim) {
                    x = kv8_in4(row + d, a.wide != 0);
                    if (d < a.c.rot && a.c.halves) {
                        const bool first = d < half;
                        const f32x4 y = kv8_in4(row + (first ? d + half : d - half), a.wide != 0);
                        const float* cs = an + 2 * (first ? d : d - half);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float re, im;
                            mmi_rope_rotate(first ? x[r] : y[r], first ? y[r] : x[r], cs[2 * r], cs[2 * r + 1], re, im);
                            x[r] = first ? re : im;
                        }
                    } else if (d < a.c.rot) {
                        const float* cs = an + d;
                        float re, im;
                        mmi_rope_rotate(x[0], x[1], cs[0], cs[1], re, im);
                        x[0] = re, x[1] = im;
                        mmi_rope_rotate(x[2], x[3], cs[2], cs[3], re, im);
                        x[2] = re, x[3] = im;
                    }
                }
                uint32_t lo[NS], hi[NS];
                kv8_split2<NS>(x[0], x[1], lo);
                kv8_split2<NS>(x[2], x[3], hi);
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    q[s][p][2 * h] = lo[s];
                    q[s][p][2 * h + 1] = hi[s];
                }
            }
        }
    }
    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = a.sink ? 0.f : -INFINITY, l = 0.f;           // (a sink of score 0 takes part in the maximum)
    for (int i = i0 + wave; i < i1; i += WK) {
        const int key0 = nb * TLM_PAGE + 16 * kq;
        const bool now = have, whole = c.whole(a.mask, nb * TLM_PAGE);
        const float sc = ks * a.mask.scale, pv = vs;
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                u32x4 lo, hi;
                C::fragments(kf[t][p], lo, hi);
#pragma unroll
                for (int n = NS - 1; n >= 0; --n) {
                    s[t] = mmi_mfma_bf16_16x16x32(lo, q[n][2 * p], s[t]);
                    s[t] = mmi_mfma_bf16_16x16x32(hi, q[n][2 * p + 1], s[t]);
                }
            }
        }
        u32x4 vw[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) vw[d] = whole ? vf[d] : kv8_quiet<E4M3>(c, a.mask, key0, vf[d]);
        load(i + WK);
        mmi_sched_barrier();
        if (!now) continue;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] *= sc;
            if (!whole)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] = c.seen(a.mask, pos, key0 + 4 * t + r) ? s[t][r] : -INFINITY;
        }
        float mx = m;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[t][r]);
        mx = mmi_rows_max(mx);
        const float ms = mx == -INFINITY ? 0.f : mx;
        if (mmi_any(mx > m)) {
            const float al = mmi_fast_exp2f(m - ms);
            l *= al;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= al;
        }
        m = mx;
        u32x4 pf[NS][2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = mmi_fast_exp2f(s[t][r] - ms);
                l += x;
                e[r] = whole || x != 0.f ? x * pv : 0.f;   // (a masked place's scale may be anything)
            }
            uint32_t lo[NS], hi[NS];
            kv8_split2<NS>(e[0], e[1], lo);
            kv8_split2<NS>(e[2], e[3], hi);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                pf[n][t >> 1][2 * (t & 1)] = lo[n];
                pf[n][t >> 1][2 * (t & 1) + 1] = hi[n];
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            u32x4 lo, hi;
            C::fragments(vw[d], lo, hi);
#pragma unroll
            for (int n = NS - 1; n >= 0; --n) {
                acc[d] = mmi_mfma_bf16_16x16x32(lo, pf[n][0], acc[d]);
                acc[d] = mmi_mfma_bf16_16x16x32(hi, pf[n][1], acc[d]);
            }
        }
    }
    l += mmi_shfl_xor(l, 16);
    l += mmi_shfl_xor(l, 32);
    if (kq == 0) {
        ml[0][wave][bl] = m;
        ml[1][wave][bl] = l;
    }
    __syncthreads();
    float M = a.sink ? 0.f : -INFINITY, L = 0.f;
#pragma unroll
    for (int v = 0; v < WK; ++v) M = fmaxf(M, ml[0][v][bl]);
    const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int v = 0; v < WK; ++v) L += ml[1][v][bl] * exp2f(ml[0][v][bl] - Ms);
    const float f = exp2f(m - Ms);
    const bool parts = a.nsplit > 1;
    const float sum = a.sink ? L + exp2f(-Ms) : L, inv = parts ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);      // (no key seen: zeros)
    const long part = ((long)slot * a.c.kv_heads + g) * a.nsplit + split;
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += 8) {
        if (d0 >= a.nd) break;
        if (d0) __syncthreads();
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (d0 + d < ND) ob[(wave * 8 + d) * 64 + lane] = acc[d0 + d < ND ? d0 + d : 0] * f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8 / WK; ++k) {
            const int d = wave + WK * k;
            if (d0 + d >= a.nd) break;
            f32x4 v = ob[d * 64 + lane];
#pragma unroll
            for (int o = 1; o < WK; ++o) v += ob[(o * 8 + d) * 64 + lane];
            v *= inv;
            if (c.c0 + bl >= c.ncol) continue;
            const int dim = (d0 + d) * 16 + 4 * kq, head = g * a.rep + col - tok * a.rep;
            if (parts) *reinterpret_cast<f32x4*>(a.po + (part * 16 + bl) * a.c.vdim + dim) = v;
            else kv8_store<Tr>(a, c.s.row0 + tok, head, dim, v);
        }
    }
    if (parts && wave == 0 && kq == 0) {
        a.pml[part * 32 + bl] = M;
        a.pml[part * 32 + 16 + bl] = L;
    }
}
template <class In, class Tr, int NS, int D, bool E4M3>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void k_tlm_kv8_attn(TlmKv8Attn a) {
    MMI_SHARED __attribute__((aligned(16))) f32x4 ob[KV8_LDS];
    MMI_SHARED float ml[2][4][16];
    tlm_kv8_attn<In, Tr, NS, D, E4M3>(a, ob, ml, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
}

// The splits of one column -> output: 16 groups of lanes take every 16th split, their sums meet in LDS.
// grid: slots of column tiles, kv heads, columns of a tile
template <class Tr>
__global__ __launch_bounds__(256) void k_tlm_kv8_combine(TlmKv8Attn a) {
    MMI_SHARED float wt[256], red[4][2];
    MMI_SHARED __attribute__((aligned(16))) f32x4 sum[256];
    const Kv8Cols c(a, (int)blockIdx.x);
    const int g = (int)blockIdx.y, bl = (int)blockIdx.z, col = c.c0 + bl, tid = (int)threadIdx.x, wave = tid >> 6;
    if (col >= c.ncol) return;
    const int ns = max(1, (c.n + a.per - 1) / a.per);      // (at most 256)
    const long part = ((long)blockIdx.x * a.c.kv_heads + g) * a.nsplit;
    float m = -INFINITY, l = 0.f;
    if (tid < ns) {
        m = a.pml[(part + tid) * 32 + bl];
        l = a.pml[(part + tid) * 32 + 16 + bl];
    }
    const float wm = mmi_wave_max_f32(m);
    if ((tid & 63) == 0) red[wave][0] = wm;
    __syncthreads();
    float M = a.sink ? 0.f : -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, red[w][0]);
    M = M == -INFINITY ? 0.f : M;
    const float w = tid < ns ? exp2f(m - M) : 0.f, wl = mmi_wave_sum_down(tid < ns ? l * w : 0.f);
    wt[tid] = w;
    if ((tid & 63) == 0) red[wave][1] = wl;
    __syncthreads();
    const float L = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]), total = a.sink ? L + exp2f(-M) : L, inv = total == 0.f ? 0.f : 1.f / total;
    const int tok = col / a.rep, head = g * a.rep + col - tok * a.rep, q = tid & 15, k = tid >> 4;
    for (int d0 = 0; d0 < a.c.vdim; d0 += 64) {
        const int d = d0 + 4 * q;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (d < a.c.vdim)
#pragma unroll 4
            for (int s = k; s < ns; s += 16) v += *(const f32x4*)(a.po + ((part + s) * 16 + bl) * a.c.vdim + d) * wt[s];
        if (d0) __syncthreads();
        sum[tid] = v;
        __syncthreads();
        if (k == 0 && d < a.c.vdim) {
#pragma unroll
            for (int i = 1; i < 16; ++i) v += sum[16 * i + q];
            kv8_store<Tr>(a, c.s.row0 + tok, head, d, v * inv);
        }
    }
}
