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
// Rows that no sequence brings.  From a sequence's end to the next one's start: all of its own, if it is passed over
template <class F>
__device__ __forceinline__ void kv8_rest_of(const TlmKv8Seqs& a, const TlmKv8Seq& s, F f) {
    const int end = mmi_uniform(kv8_row0(a, s.e + 1));
    for (int i = s.row0 + s.len; i < end; ++i) f(i);
}
// Before the first sequence and behind the last one, which may be most rows of a padded call: shared by all workgroups, `n` (of 8000 rows
// of 32 heads of 128, 100 brought: 68 us, 49 of it the attention itself; by one workgroup for each kv head 994)
template <class F>
__device__ __forceinline__ void kv8_rest_around(const TlmKv8Seqs& a, int first, int n, F f) {
    if (!a.row0) return;
    const int head = mmi_uniform(kv8_row0(a, 0)), tail = mmi_uniform(kv8_row0(a, a.n));
    for (int i = first; i < head + a.T - tail; i += n) f(i < head ? i : tail + i - head);
}
// page number of the sequence's tokens 64 i .. 64 i + 63; -1: there is none
__device__ __forceinline__ int kv8_page(const TlmKv8Seqs& a, int n_pages, const int* row, int i) {
    if (!a.ring && i >= a.pages.ld) return -1;
    const int p = row[a.ring && i >= a.pages.keep ? a.pages.keep + (i - a.pages.keep) % (a.pages.ld - a.pages.keep) : i];
    return p < 0 || p >= n_pages ? -1 : p;
}
__device__ __forceinline__ const int* kv8_table(const TlmKv8Seqs& a, int e) { return a.pages.table + (long)mmi_uniform(a.slot ? a.slot[e] : e) * a.pages.ld; }

// An entry's work is cut into pieces of `per` units, `mul` units a row, without anyone having counted them: entry e owns the slots from
// row0[e] * mul / per + extra e on, which are as many as it can need, and a slot's entry is the last one that begins at or before it.
// (by > 0: only entries with at least `by` units need a slot; one more for each `by` units is then enough, where that is fewer than one per entry.)
struct Kv8Cut { int mul, per, extra, by; };            // mul 0: `extra` slots per entry
MMI_HD int kv8_slots_before(const Kv8Cut& z, int row, int e) {
    const unsigned u = (unsigned)row * (unsigned)z.mul;    // (below 2^31; `per` is a power of two)
    return (int)(u >> __builtin_ctz(z.per)) + (z.by ? (int)(u / (unsigned)z.by) : z.extra * e);
}
__device__ __forceinline__ int kv8_slot0(const TlmKv8Seqs& a, const Kv8Cut& z, int e) { return z.mul ? kv8_slots_before(z, kv8_row0(a, e), e) : z.extra * e; }
__device__ __forceinline__ int kv8_find(const TlmKv8Seqs& a, const Kv8Cut& z, int slot) {
    if (!z.mul) return min(slot / z.extra, a.n - 1);
    unsigned below = 0;
    for (int e = mmi_lane(); e < a.n; e += 64) below += kv8_slot0(a, z, e) <= slot ? 1u : 0u;
    return max(mmi_uniform((int)mmi_wave_sum_u32(below) - 1), 0);
}
// host: the cut of mul * rows units (one row each: nothing to look for), and how many slots there are
inline Kv8Cut kv8_cut(const TlmKv8Seqs& a, int mul, int per, int more) { return a.row0 ? Kv8Cut{mul, per, more, 0} : Kv8Cut{0, per, mmi_cdiv(mul, per), 0}; }
inline long kv8_slots(const TlmKv8Seqs& a, const Kv8Cut& z) { return z.mul ? kv8_slots_before(z, a.T, a.n) + (z.by ? 1 : 0) : (long)z.extra * a.n; }

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
    static __device__ __forceinline__ u32x2 f16(uint32_t w) { return E4M3 ? mmi_fp8x4_to_f16(w) : mmi_i8x4_to_f16(w); }
    // 16 codes -> two operand fragments of 8
    static __device__ __forceinline__ void fragments(u32x4 c, u32x4& lo, u32x4& hi) {
        const u32x2 a = f16(c[0]), b = f16(c[1]), d = f16(c[2]), e = f16(c[3]);
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
// dimensions d .. d + 3 (d a multiple of 4) turned (cs: the position's angles; y: the partners, where these lie half of the dimensions apart)
__device__ __forceinline__ f32x4 kv8_turned4(const TlmKv8Cache& c, f32x4 x, f32x4 y, int d, const float* cs) {
    if (d >= c.rot) return x;
    if (c.halves) {
        const bool first = d < c.rot / 2;
        cs += 2 * (first ? d : d - c.rot / 2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float re, im;
            mmi_rope_rotate(first ? x[r] : y[r], first ? y[r] : x[r], cs[2 * r], cs[2 * r + 1], re, im);
            x[r] = first ? re : im;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            float re, im;
            mmi_rope_rotate(x[r], x[r + 1], cs[d + r], cs[d + r + 1], re, im);
            x[r] = re;
            x[r + 1] = im;
        }
    }
    return x;
}
template <class In>
__device__ __forceinline__ f32x4 kv8_partners4(const TlmKv8Cache& c, const In* row, int d, bool wide) {
    const int rot = c.halves ? c.rot : 0, half = rot / 2;
    return d < rot ? kv8_in4(row + (d < half ? d + half : d - half), wide) : f32x4{0.f, 0.f, 0.f, 0.f};
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
struct Kv8Span { TlmKv8Seq s; int page, part, lo, hi, row, pos; bool none, first; };
__device__ __forceinline__ Kv8Span kv8_span(const TlmKv8Seqs& q, const Kv8Cut& z, int n_pages, int slot) {
    const int e = kv8_find(q, z, slot);
    const TlmKv8Seq s = kv8_seq(q, e);
    const int i = slot - kv8_slot0(q, z, e), b = s.pos0 / KV8_BLOCK + i;      // block of the sequence
    Kv8Span o;
    o.s = s;
    o.first = i == 0;
    o.pos = b * KV8_BLOCK;
    o.none = s.len < 1 || i < 0 || o.pos >= s.pos0 + s.len;      // (i < 0: row starts that do not ascend)
    o.lo = max(s.pos0 - o.pos, 0);
    o.hi = min(s.pos0 + s.len - o.pos, KV8_BLOCK);
    o.row = s.row0 + o.pos - s.pos0;               // row of the block's first token (of token lo on they are the call's)
    o.page = o.none ? -1 : kv8_page(q, n_pages, kv8_table(q, e), b / KV8_PARTS);
    o.part = b % KV8_PARTS;
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

// Four elements as they come, to be widened behind the last load: a conversion beside each load would wait for it, 18 us for the values of a
// block of prompts where all of it together takes 4.
template <class In> struct Kv8In;
template <> struct Kv8In<float> {
    typedef f32x4 T;
    static __device__ __forceinline__ T slow(const float* p) { return T{p[0], p[1], p[2], p[3]}; }
    static __device__ __forceinline__ f32x4 wide(T x) { return x; }
    static __device__ __forceinline__ float wide(float x) { return x; }
};
template <> struct Kv8In<uint16_t> {
    typedef u32x2 T;
    static __device__ __forceinline__ T slow(const uint16_t* p) { return T{p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16}; }
    static __device__ __forceinline__ f32x4 wide(T w) {
        return f32x4{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16),
                     __builtin_bit_cast(float, w[1] & 0xffff0000u)};
    }
    static __device__ __forceinline__ float wide(uint16_t x) { return mmi_bf16_to_f32(x); }
};
// the first n of four bytes
__device__ __forceinline__ uint32_t kv8_bytes_below(int n) { return n <= 0 ? 0u : (n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u); }
// pair p's angle at a position, where its dimensions find it
__device__ __forceinline__ void kv8_put_angle(const TlmKv8Cache& c, float* cs, float* sn, int pos, int p, double freq) {
    float co, si;
    kv8_angle(pos, freq, co, si);
    const int d = c.halves ? p : 2 * p, e = c.halves ? p + c.rot / 2 : d + 1;
    cs[d] = cs[e] = co;
    sn[d] = -si;
    sn[e] = si;
}
// One wave per block, head and side; four heads a workgroup, which form the angles of the block's tokens once.  A few tokens' call is as long as its
// chain of loads and its code's way to the CU, so no load waits for another that it does not need, nothing branches around one (lanes without a
// token of the call read its nearest), and the common path is short.
// grid: slots of blocks, kv heads / 4, 2 (keys, values)
//   keys: four lanes per token, granules of 4 dimensions in turn      values: a lane per dimension, its 16 tokens side by side
// Measured (8 heads of 128, bf16): 3.6k tokens in three portions 13 us for 25 MB, the rest latency; one token 5.8 us, 64 tokens 7.0 us, of which an
// empty launch is 1.4.  Heads of up to 128 dimensions have an instance of their own (68 registers; as the one for 256, 117 and half the waves on a CU).
template <class In, bool E4M3, int D>
__global__ __launch_bounds__(256, D == 128 ? 4 : 2) void k_tlm_kv8_append(TlmKv8Append a) {
    typedef Kv8Code<E4M3> C;
    typedef Kv8In<In> R;
    constexpr int N = D / 16, LD = D + 16;                 // granules of a lane; floats of a token's angles (two tokens' reads: banks of their own)
    MMI_SHARED float cs[KV8_BLOCK * LD], sn[KV8_BLOCK * LD];      // [token][dimension]: cosine; sine, with the sign that the partner takes
    const Kv8Span s = kv8_span(a.q, a.z, a.c.n_pages, (int)blockIdx.x);
    if (s.none) return;                                    // (the page is looked at behind the first loads: it is on its way meanwhile)
    const int lane = mmi_lane(), g = (int)blockIdx.y * 4 + mmi_uniform((int)threadIdx.x >> 6), gc = min(g, a.c.kv_heads - 1);
    const bool held = s.lo > 0;
    const long unit = (long)s.page * a.c.kv_heads + gc;
    if (blockIdx.z == 0) {
        const int t = lane >> 2, c = lane & 3, n = a.c.dim / 16, rot = a.c.rot, half = rot / 2;
        const In* row = (const In*)a.k + (long)(s.row + min(max(t, s.lo), s.hi - 1)) * a.k_row + (long)gc * a.k_head;
        typename R::T x[N], y[N];
        auto at = [&](int i) { return 4 * (c + 4 * min(i, n - 1)); };
        auto partner = [&](int d) { return d < half ? d + half : (d < rot ? d - half : d); };
        if (a.wide) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const typename R::T*)(row + at(i));
            if (rot && a.c.halves) {
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = *(const typename R::T*)(row + partner(at(i)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = R::slow(row + at(i));
                y[i] = R::slow(row + partner(at(i)));
            }
        }
        if (s.page < 0) return;
        uint32_t* out = (uint32_t*)(a.c.k + (unit * TLM_PAGE + s.part * KV8_BLOCK + t) * a.c.dim);
        float* scale = a.c.ks + unit * KV8_PARTS + s.part, ratio;
        const float before = held ? *scale : 0.f;
        uint32_t old[N];
        if (held) {
#pragma unroll
            for (int i = 0; i < N; ++i) old[i] = out[at(i) / 4];
        }
        if (rot) {
            const int step = 256 / half, all = (s.hi - s.lo) * half;      // (half is at most 128)
            int u = (int)threadIdx.x / half, p = (int)threadIdx.x % half;
            if (step * half == 256) {                                     // a thread's pair stays the same
                const double freq = a.c.freq[p];
                for (; u < s.hi - s.lo; u += step) kv8_put_angle(a.c, cs + (s.lo + u) * LD, sn + (s.lo + u) * LD, s.pos + s.lo + u, p, freq);
            } else {
                for (int i = (int)threadIdx.x; i < all; i += 256) {
                    u = s.lo + i / half;
                    p = i % half;
                    kv8_put_angle(a.c, cs + u * LD, sn + u * LD, s.pos + u, p, a.c.freq[p]);
                }
            }
            __syncthreads();
        }
        const bool fresh = t >= s.lo && t < s.hi;
        f32x4 z[N];
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            z[i] = R::wide(x[i]);
            if (rot) {
                const f32x4 o = R::wide(y[i]), w = a.c.halves ? o : f32x4{z[i][1], z[i][0], z[i][3], z[i][2]};
                const f32x4 co = *(const f32x4*)(cs + t * LD + at(i)), si = *(const f32x4*)(sn + t * LD + at(i));
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float turned = mmi_fma(w[r], si[r], z[i][r] * co[r]);
                    z[i][r] = at(i) < rot ? turned : z[i][r];
                }
            }
            bits = max(bits, kv8_bits(z[i]));
        }
        bits = mmi_wave_max_u32(fresh ? bits : 0u);
        if (g >= a.c.kv_heads) return;
        const float after = kv8_grown<E4M3>(before, held, bits, ratio), inv = 1.f / after;
        const bool bad = !(after == after);
        if (fresh) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) out[c + 4 * i] = bad ? 0u : C::pack(z[i] * inv);
        } else if (t < s.lo && ratio != 1.f) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) out[c + 4 * i] = bad ? 0u : C::pack(C::unpack(old[i]) * ratio);
        }
        if (lane == 0) *scale = after;
    } else {
        const In* v = (const In*)a.v + (long)s.row * a.v_row + (long)gc * a.v_head;
        In x[D / 64][KV8_BLOCK];
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int t = 0; t < KV8_BLOCK; ++t) x[i][t] = v[(long)min(max(t, s.lo), s.hi - 1) * a.v_row + min(lane + 64 * i, a.c.vdim - 1)];
        if (s.page < 0 || g >= a.c.kv_heads) return;
        const bool whole = s.lo == 0 && s.hi == KV8_BLOCK;
        u32x4* out = (u32x4*)(a.c.v + unit * a.c.vdim * TLM_PAGE + s.part * KV8_BLOCK);
        auto at = [&](int i) { return min(lane + 64 * i, a.c.vdim - 1) * (TLM_PAGE / 16); };
        float* scale = a.c.vs + unit * KV8_PARTS + s.part, ratio;
        const float before = held ? *scale : 0.f;
        u32x4 old[D / 64];
        if (!whole) {                                      // (the bytes behind the last token stay what they are)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) old[i] = out[at(i)];
        }
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int t = 0; t < KV8_BLOCK; ++t) bits = max(bits, __builtin_bit_cast(unsigned, R::wide(x[i][t])) & 0x7fffffffu);
        bits = mmi_wave_max_u32(bits);
        const float after = kv8_grown<E4M3>(before, held, bits, ratio), inv = 1.f / after;
        const bool bad = !(after == after);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 y = {R::wide(x[i][4 * j]), R::wide(x[i][4 * j + 1]), R::wide(x[i][4 * j + 2]), R::wide(x[i][4 * j + 3])};
                w[j] = bad ? 0u : C::pack(y * inv);
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b = old[i][j], was = bad ? 0u : (ratio != 1.f ? C::pack(C::unpack(b) * ratio) : b);
                    const uint32_t o = kv8_bytes_below(s.lo - 4 * j), m = kv8_bytes_below(s.hi - 4 * j) & ~o;      // tokens held, new ones
                    w[j] = (w[j] & m) | (was & o) | (b & ~(m | o));
                }
            }
            if (lane + 64 * i < a.c.vdim) out[at(i)] = w;
        }
        if (lane == 0) *scale = after;
    }
}

// ---- read: the values that the cache holds for the call's rows --------------------------------------------------------------
struct TlmKv8Read {
    TlmKv8Cache c;
    TlmKv8Seqs q;
    Kv8Cut z;
    void *k, *v;                         // [rows][kv heads][dim], [rows][kv heads][vdim]; tokens without a page, rows without a sequence: zeros
};
__device__ __forceinline__ void kv8_put4(float* p, f32x4 v) { TlmF32::store4(p, v); }
__device__ __forceinline__ void kv8_put4(uint16_t* p, f32x4 v) { TlmBf16::store4(p, v); }
__device__ __forceinline__ void kv8_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void kv8_put(uint16_t* p, float v) { *p = mmi_f32_to_bf16(v); }
// Eight loads a lane on their way, then stores: 3.6k tokens of 8 heads of 128 in bf16 11 us for 25 MB, 64 tokens 7 us (positions, page, codes: a chain).
// grid: slots of blocks, kv heads, 2
template <class Out, bool E4M3>
__global__ __launch_bounds__(64) void k_tlm_kv8_read(TlmKv8Read a) {
    typedef Kv8Code<E4M3> C;
    const Kv8Span s = kv8_span(a.q, a.z, a.c.n_pages, (int)blockIdx.x);
    const int lane = mmi_lane(), g = (int)blockIdx.y;
    auto clear = [&](int row) __attribute__((always_inline)) {
        const int n = blockIdx.z ? a.c.vdim : a.c.dim;
        if (4 * lane < n) kv8_put4((Out*)(blockIdx.z ? a.v : a.k) + ((long)row * a.c.kv_heads + g) * n + 4 * lane, f32x4{0.f, 0.f, 0.f, 0.f});
    };
    kv8_rest_around(a.q, (int)blockIdx.x, (int)gridDim.x, clear);
    if (s.first) kv8_rest_of(a.q, s.s, clear);
    if (s.none) return;
    const bool lost = s.page < 0;
    const long unit = (long)max(s.page, 0) * a.c.kv_heads + g;
    const float scale = lost ? 0.f : (blockIdx.z ? a.c.vs : a.c.ks)[unit * KV8_PARTS + s.part];
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (blockIdx.z == 0) {
        const int t = lane >> 2, c = lane & 3;
        if (t < s.lo || t >= s.hi) return;
        const uint32_t* in = (const uint32_t*)(a.c.k + (unit * TLM_PAGE + s.part * KV8_BLOCK + t) * a.c.dim);
        Out* out = (Out*)a.k + ((long)(s.row + t) * a.c.kv_heads + g) * a.c.dim;
        const int n = a.c.dim / 16;
        for (int i0 = 0; i0 < n; i0 += 8) {                // (eight loads on their way at once)
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = in[c + 4 * min(i0 + i, n - 1)];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + i < n) kv8_put4(out + 4 * (c + 4 * (i0 + i)), lost ? zero : C::unpack(w[i]) * scale);
        }
    } else {
        const u32x4* in = (const u32x4*)(a.c.v + unit * a.c.vdim * TLM_PAGE + s.part * KV8_BLOCK);
        const long ld = (long)a.c.kv_heads * a.c.vdim;
        for (int d0 = lane; d0 < a.c.vdim; d0 += 128) {
            u32x4 w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = in[min(d0 + 64 * i, a.c.vdim - 1) * (TLM_PAGE / 16)];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = d0 + 64 * i;
                if (d >= a.c.vdim) break;
                Out* out = (Out*)a.v + ((long)s.row * a.c.kv_heads + g) * a.c.vdim + d;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 x = lost ? zero : C::unpack(w[i][j]) * scale;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (4 * j + r >= s.lo && 4 * j + r < s.hi) kv8_put(out + (4 * j + r) * ld, x[r]);
                }
            }
        }
    }
}

// ---- attention -----------------------------------------------------------------------------------------------------------
// Numerics, both kernels.  Operands are fp16, 11 bits: codes are exact in it, queries are first brought to [2^14, 2^15) by a power of two of
// their own, softmax weights are carried times the value scale of their block.  Two running references, powers of two both (moving one rounds
// nothing): r of the scores, which weights and their sum are relative to, and r + off of score + exponent of the value scale, which weights times
// scale are relative to.  So what the products take lies between 2^7 and 2^15 at its largest, however blocks' scales differ, and the denominator does not
// know of the scales: blocks of zeros, whose scale is 2^-107, neither let it overflow nor are lost from it beside values of 2^20.  References, with
// the sums, move only where a maximum has outgrown one by 2^6.  One fp16 rounding (2^-12) is below a bf16 result's own; for fp32 queries both
// operands come in two parts, 22 bits, good to 2^-24.  (bf16 operands left 1.8 times the error of the result's rounding.)  Sums, maxima and the
// denominator, which has the weights before they were rounded, are fp32.
// Sequences with up to so many columns, one tile, are the few's where a call may bring longer ones: 64 sequences with 4 rows of 4 heads, 2000 keys each,
// take 52 us there and 101 us as the many's; 2 with 20 000 keys, 27 and 46 us.  (A second tile would read every key again.)
constexpr int KV8_FEW = 16;
constexpr int KV8_MANY = 128;            // columns of a workgroup of the many's
constexpr float KV8_UP = 8.f, KV8_SLACK = 6.f;      // log2: of what weights are carried times, of what they may outgrow it by (fp16 ends at 2^16)
constexpr int KV8_ANGLES = 2048;         // pairs of a cosine and a sine in LDS

struct Kv8Share {                        // one kernel's part of a call
    Kv8Cut z;                            // of columns (token, head of the group), by groups of z.per
    int cols;                            // columns that a slot can have: z.per, or fewer where no group has more
    int pages, nsplit;                   // pages per split; splits that a group can need
    float* po;                           // nsplit > 1: [group slot][kv head][split][z.per columns][vdim] results of the split alone, without the sink
    float* pml;                          // [group slot][kv head][split][2][z.per]: reference of the scores, sum of weights
    int* what;                           // [group slot][4]: its columns, the splits that were needed, first row and column of its sequence
};
struct TlmKv8Attn {
    TlmKv8Cache c;
    TlmKv8Seqs q;
    const void* x; long x_row, x_head;   // queries
    int wide;                            // every 4 of their elements are aligned
    void* out; long out_row, out_head;   // rows; out_ks > 0: fragment-packed rows (tlm_index), columns head * 16 nd + d
    int out_ks;
    int rep, nd;                         // query heads per key/value head; vdim / 16
    TlmMask mask;                        // scale: log2 e times the softmax's
    int sink;                            // one is added to the denominator
    int rest;                            // rows that no sequence brings become zeros
    int both;                            // sequences of more than KV8_FEW columns are `many`'s; otherwise all are `few`'s
    Kv8Share few, many;
};

// columns c0 .. c0 + per - 1 of one entry, and the pages that they see: [0, n0) and [b0, b0 + n - n0)
struct Kv8Cols {
    TlmKv8Seq s;
    int c0, ncol, plo, phi, n0, b0, n;
    __device__ __forceinline__ Kv8Cols(const TlmKv8Attn& a, const Kv8Share& h, bool few, int slot) {
        const int e = kv8_find(a.q, h.z, slot), per = h.z.per;
        s = kv8_seq(a.q, e);
        c0 = (slot - kv8_slot0(a.q, h.z, e)) * per;
        ncol = s.len * a.rep;
        plo = phi = n = n0 = b0 = 0;
        if (c0 < 0) c0 = ncol = 0;                         // (row starts that do not ascend)
        if (a.both && (ncol <= KV8_FEW) != few) ncol = 0;
        if (c0 >= ncol) return;
        plo = s.pos0 + c0 / a.rep;
        phi = s.pos0 + min(c0 + per - 1, ncol - 1) / a.rep;
        const int w = a.mask.window;
        b0 = w > 0 && plo - w + 1 > 0 ? (plo - w + 1) / TLM_PAGE : 0;
        n0 = w > 0 ? min(b0, (a.mask.keep + TLM_PAGE - 1) / TLM_PAGE) : 0;
        if (!a.q.ring) n0 = min(n0, a.q.pages.ld);
        n = n0 + phi / TLM_PAGE + 1 - b0;
        if (!a.q.ring) n = min(n, n0 + max(a.q.pages.ld - b0, 0));      // (so that the splits, as many as a sequence of `ld` pages needs, are enough)
    }
    __device__ __forceinline__ int page(int i) const { return i < n0 ? i : b0 + i - n0; }
};
// The pages of a walk, 64 of them a load, a lane each: what a step's page is comes out of a register (a scalar load per step is a wait of its
// own, and one for every LDS read in flight).  Asked for in ascending order.
struct Kv8Pages {
    int held, from;
    __device__ __forceinline__ void fill(const TlmKv8Attn& a, const Kv8Cols& c, const int* bt, int i) {
        from = i;
        const int k = min(i + mmi_lane(), c.n - 1), p = c.page(max(k, 0));
        held = kv8_page(a.q, a.c.n_pages, bt, p);
    }
    __device__ __forceinline__ int at(const TlmKv8Attn& a, const Kv8Cols& c, const int* bt, int i) {
        if (i >= from + 64) fill(a, c, bt, i);
        return mmi_from_lane(held, i - from);
    }
};
// for the kernel that joins the splits, which would have to look for it in every wave (of 64 sequences with 4 rows each, 20 us for slots without a column)
__device__ __forceinline__ void kv8_tell(const Kv8Share& h, const Kv8Cols& c, int slot, int g, int split) {
    if (h.nsplit > 1 && g == 0 && split == 0 && threadIdx.x == 0)
        *(u32x4*)(h.what + 4 * slot) = u32x4{(unsigned)max(0, c.ncol - c.c0), (unsigned)max(1, (c.n + h.pages - 1) / h.pages), (unsigned)c.s.row0, (unsigned)c.c0};
}
// exponent of a value scale as it is stored, 127 for [1, 2); at least 27: what lies below 2^-100 fits into the weights' 2^7 and more
__device__ __forceinline__ float kv8_exponent(float scale) { return (float)max(__builtin_bit_cast(unsigned, scale) >> 23 & 255u, 27u); }
// A column's references: r = ceil(maximum of the scores) when it was moved last, off the same of score - r + exponent of the value scale.
struct Kv8Refs {
    static constexpr float LEAST = -3.4028234663852886e38f, NONE = -1024.f;      // nothing has been seen (finite, so that differences are numbers)
    float r = LEAST, off = NONE;
    float up = 0.f;                      // 2^(KV8_UP + 127 - off): weights times value scale times this are the product's operand
    // does a lane's maximum `top` of scores in a block of exponent e outgrow one of them?
    __device__ __forceinline__ bool outgrown(float top, float e) const { return top - r + fmaxf(e - off, 0.f) > KV8_SLACK; }
    // moved to the column's maxima (max over its lanes: `across`); factors of the sum of weights and of the weighted sums
    template <class F>
    __device__ __forceinline__ void move(float top, float e, F across, float& fewer, float& less) {
        const float to = fmaxf(r, ceilf(across(top))), held = off - (to - r), out = fmaxf(held, ceilf(across(top - to + e)));
        fewer = mmi_fast_exp2f(r - to);
        less = mmi_fast_exp2f(held - out);
        r = to;
        off = out;
        up = mmi_fast_exp2f(KV8_UP + 127.f - off);
    }
    // what a block's weights are multiplied by: its scale and `up` (where that leaves fp32, all of its weights are below 2^-100 of the largest); a block that
    // the column does not see may have any scale
    __device__ __forceinline__ float times(float scale, float top) const {
        const float x = scale * up;
        return top == -INFINITY ? 0.f : (fabsf(x) > 0x1p126f ? 0x1p126f : x);
    }
};
// scores of keys key0 .. key0 + 15 for a query at `pos`, -infinity where it does not see them
__device__ __forceinline__ void kv8_masked(const TlmMask& m, int pos, int key0, float (&y)[16]) {
    const int behind = m.window > 0 ? pos - m.window : -1;      // the last position that a window has passed
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = (key0 + r <= pos) & ((key0 + r > behind) | (key0 + r < m.keep)) ? y[r] : -INFINITY;
}
// positions plo .. phi all see the n keys from key0 on
__device__ __forceinline__ bool kv8_whole(const TlmMask& m, int plo, int phi, int key0, int n) { return key0 + n - 1 <= plo && (m.window <= 0 || phi - key0 < m.window || key0 + n <= m.keep); }

// e4m3 bytes of tokens that no column sees may hold anything, a NaN among it, which a weight of zero would not silence: cleared
template <bool E4M3>
__device__ __forceinline__ u32x4 kv8_quiet(const Kv8Cols& c, const TlmMask& m, int key0, u32x4 w) {
    if constexpr (!E4M3) return w;
    const int behind = m.window > 0 ? c.plo - m.window : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t keep = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = key0 + 4 * j + r;
            keep |= (key <= c.phi) & ((key > behind) | (key < m.keep)) ? 0xffu << (8 * r) : 0u;
        }
        w[j] &= keep;
    }
    return w;
}

// fp32 -> NS parts of fp16, pairs packed
template <int NS>
__device__ __forceinline__ void kv8_split2(float a, float b, uint32_t (&o)[NS]) {
    o[0] = mmi_pack_f16x2(a, b);
    if constexpr (NS == 2) {
        const f32x2 h = mmi_unpack_f16x2(o[0]);
        o[1] = mmi_pack_f16x2(a - h[0], b - h[1]);
    }
}
template <int NS>
__device__ __forceinline__ void kv8_split8(const float* x, float f, u32x4 (&q)[NS]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t o[NS];
        kv8_split2<NS>(x[2 * j] * f, x[2 * j + 1] * f, o);
#pragma unroll
        for (int s = 0; s < NS; ++s) q[s][j] = o[s];
    }
}
// the power of two that brings `amax` to [2^14, 2^15), and its inverse (limits: 2^-100 and what is not finite)
__device__ __forceinline__ float kv8_raise(float amax, float& back) {
    const int e = max((int)(__builtin_bit_cast(unsigned, amax) >> 23) - 127, -100);
    back = __builtin_bit_cast(float, (unsigned)(min(e, 127) - 14 + 127) << 23);
    return __builtin_bit_cast(float, (unsigned)(14 - min(e, 127) + 127) << 23);
}
// a lane's 8 dimensions of a query row, and their rotation partners where these lie half of the dimensions apart
struct Kv8Raw { f32x4 x[2], y[2]; };
template <class In>
__device__ __forceinline__ Kv8Raw kv8_raw(const TlmKv8Attn& a, const In* row, int d) {
    const bool wide = a.wide != 0;
    Kv8Raw o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int e = d + 4 * h;
        o.x[h] = e < a.c.dim ? kv8_in4(row + e, wide) : f32x4{0.f, 0.f, 0.f, 0.f};
        o.y[h] = kv8_partners4(a.c, row, e, wide);
    }
    return o;
}
// The group's queries into LDS as operand fragments, by the whole workgroup: D / 8 lanes a column, and a token's angles formed once for all
// heads (a portion of the tokens at a time).  put(column, 8 dimensions d / 8 .., part): where they go; back: the columns' inverse factors.
template <class In, int NS, int D, class Put>
__device__ __forceinline__ void kv8_queries(const TlmKv8Attn& a, const Kv8Cols& c, int per, int g, float* angle, float* back, Put put) {
    constexpr int G = D / 8, AT = 256 / G;                 // lanes a column, columns at a time
    const int tid = (int)threadIdx.x, half = a.c.rot / 2, cols = min(per, c.ncol - c.c0), t1 = (c.c0 + cols - 1) / a.rep;
    const int tokens = half ? KV8_ANGLES / half : t1 + 1;  // (half is 128 at most)
    for (int t0 = c.c0 / a.rep; t0 <= t1; t0 += tokens) {
        const int nt = min(tokens, t1 - t0 + 1), n0 = max(0, t0 * a.rep - c.c0), n1 = min(cols, (t0 + nt) * a.rep - c.c0);
        if (half) {
            __syncthreads();
            for (int i = tid; i < nt * half; i += 256) kv8_angle(c.s.pos0 + t0 + i / half, a.c.freq[i % half], angle[2 * i], angle[2 * i + 1]);
            __syncthreads();
        }
        // four rounds of columns are asked for at once; every lane goes along, the maximum is taken across them
        for (int nb = n0; nb < n1; nb += 4 * AT) {
            Kv8Raw raw[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int col = c.c0 + min(nb + u * AT + tid / G, n1 - 1), tok = col / a.rep;
                if (nb + u * AT < n1) raw[u] = kv8_raw(a, (const In*)a.x + (long)(c.s.row0 + tok) * a.x_row + (g * a.rep + col - tok * a.rep) * a.x_head, 8 * (tid % G));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (nb + u * AT >= n1) break;
                const int n = nb + u * AT + tid / G, k = min(n, n1 - 1), tok = (c.c0 + k) / a.rep, d = 8 * (tid % G);
                float x[8], top = 0.f, b;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = kv8_turned4(a.c, raw[u].x[h], raw[u].y[h], d + 4 * h, angle + (tok - t0) * 2 * half);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[4 * h + r] = v[r];
                        top = fmaxf(top, fabsf(v[r]));
                    }
                }
                u32x4 q[NS];
                kv8_split8<NS>(x, kv8_raise(mmi_group_max<G>(top), b), q);
                if (n < n1) {
#pragma unroll
                    for (int s = 0; s < NS; ++s) *put(k, tid % G, s) = q[s];
                    if (tid % G == 0) back[k] = b;
                }
            }
        }
    }
    __syncthreads();
}
// four dimensions of a row's head
template <class Tr>
__device__ __forceinline__ void kv8_store(const TlmKv8Attn& a, int row, int head, int d, f32x4 v) {
    typedef typename Tr::elem E;
    Tr::store4((E*)a.out + (a.out_ks ? tlm_index<Tr>(row, head * 16 * a.nd + d, a.out_ks) : row * a.out_row + head * a.out_head + d), v);
}
// zeros for a group's heads of a row
template <class Tr>
__device__ __forceinline__ void kv8_clear(const TlmKv8Attn& a, int row, int g) {
    const int d = 4 * ((int)threadIdx.x & 63);
    for (int head = (int)threadIdx.x >> 6; head < a.rep; head += 4)
        if (d < a.c.vdim) kv8_store<Tr>(a, row, g * a.rep + head, d, f32x4{0.f, 0.f, 0.f, 0.f});
}
// 1 / denominator of weights that were summed relative to 2^r; nothing seen: zero
__device__ __forceinline__ float kv8_inverse(float L, float r, int sink) {
    const float sum = sink ? L + exp2f(-r) : L;
    return sum == 0.f ? 0.f : 1.f / sum;
}

// Few columns: four waves share one tile of 16 columns, each takes every fourth of its pages straight from the cache - the page after it is
// asked for before the products of this one - and their sums meet in LDS.  Bound by the codes' way from memory: 100 003 keys of 8 heads of 128
// 38.8 us at 5.3 TB/s, as fast as a large copy; 64 sequences of 800 to 4096 keys 76 us at 4.2 TB/s, the longest ones' end is not full.
// LDS: the queries and their angles, then (the same memory) the waves' sums
constexpr int KV8_LDS = 4 * 8 * 64;                        // vectors of four floats: 8 waves' worth of 8 x 16 dimensions; queries of 256 in two parts and angles take 2048 too
template <class In, class Tr, int NS, int D, bool E4M3>
__device__ __forceinline__ void tlm_kv8_attn(const TlmKv8Attn& a, f32x4* ob, float (*ml)[4][16], int slot, int g, int split) {
    typedef Kv8Code<E4M3> C;
    constexpr int NP = D / 64, ND = D / 16, WK = 4;
    const int lane = (int)threadIdx.x & 63, wave = mmi_uniform((int)threadIdx.x >> 6), bl = lane & 15, kq = lane >> 4;
    const Kv8Cols c(a, a.few, true, slot);
    kv8_tell(a.few, c, slot, g, split);
    if (a.rest && split == 0 && c.c0 == 0 && c.s.len == 0) kv8_rest_of(a.q, c.s, [&](int row) __attribute__((always_inline)) { kv8_clear<Tr>(a, row, g); });
    const int i0 = split * a.few.pages, i1 = min(c.n, i0 + a.few.pages);
    if (c.c0 >= c.ncol || (i0 >= i1 && split > 0)) return;
    const int col = min(c.c0 + bl, c.ncol - 1), tok = col / a.rep, pos = c.s.pos0 + tok;
    const bool live = c.c0 + bl < c.ncol;
    const int* bt = kv8_table(a.q, c.s.e);
    u32x4 kf[4][NP], vf[ND];
    float ks = 0.f, vs = 0.f;
    int nb = 0;
    bool have = false;
    Kv8Pages pages;
    pages.fill(a, c, bt, i0);
    // (past the end, and where there is no page: the pool's first one, unused)
    auto load = [&](int i) __attribute__((always_inline)) {
        i = min(i, i1 - 1);
        nb = c.page(i);
        const int p = pages.at(a, c, bt, i);
        have = p >= 0;
        const long unit = (long)max(p, 0) * a.c.kv_heads + g;
        const uint8_t* kp = a.c.k + (unit * TLM_PAGE + 16 * (bl >> 2) + (bl & 3)) * a.c.dim;
        const uint8_t* vp = a.c.v + (unit * a.c.vdim + bl) * TLM_PAGE + 16 * kq;
        ks = a.c.ks[unit * KV8_PARTS + kq];
        vs = a.c.vs[unit * KV8_PARTS + kq];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) kf[t][p] = mmi_load_nt((const u32x4*)(kp + 4 * t * a.c.dim + (64 * p + 16 * kq < a.c.dim ? 64 * p + 16 * kq : 0)));      // (dimensions past the head's meet zeros)
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[d] = mmi_load_nt((const u32x4*)(vp + min(d, a.nd - 1) * 16 * TLM_PAGE));
    };
    if (i0 + wave < i1) load(i0 + wave);
    u32x4* qf = reinterpret_cast<u32x4*>(ob);              // fragments [p][part]: dimensions 64 (p / 2) + 16 kq + 8 (p & 1) ..
    kv8_queries<In, NS, D>(a, c, 16, g, reinterpret_cast<float*>(ob + 2 * NP * NS * 64), &ml[0][0][0], [&](int n, int k, int s) __attribute__((always_inline)) {
        return qf + ((2 * (k >> 3) + (k & 1)) * NS + s) * 64 + 16 * ((k >> 1) & 3) + n;
    });
    u32x4 q[2 * NP][NS];
#pragma unroll
    for (int p = 0; p < 2 * NP; ++p)
#pragma unroll
        for (int s = 0; s < NS; ++s) q[p][s] = qf[(p * NS + s) * 64 + lane];
    float back = ml[0][0][bl];
    __syncthreads();                                       // (their memory takes the sums)
    back *= a.mask.scale;
    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    Kv8Refs ref;
    float l = 0.f;
    for (int i = i0 + wave; i < i1; i += WK) {
        const int key0 = nb * TLM_PAGE + 16 * kq;
        const bool now = have, whole = kv8_whole(a.mask, c.plo, c.phi, nb * TLM_PAGE, TLM_PAGE);
        const float sc = ks * back, vsn = vs;
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
                    s[t] = mmi_mfma_f16_16x16x32(lo, q[2 * p][n], s[t]);
                    s[t] = mmi_mfma_f16_16x16x32(hi, q[2 * p + 1][n], s[t]);
                }
            }
        }
        u32x4 vw[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) vw[d] = whole ? vf[d] : kv8_quiet<E4M3>(c, a.mask, key0, vf[d]);
        load(i + WK);
        mmi_sched_barrier();
        if (!now) continue;
        // (Scalars, changed in selects: where elements of s were changed one at a time behind `if (!whole)` while it lived in accumulation registers, the
        // compiler wrote its first element over the others on that path.  What is changed behind branches here, acc, is changed whole.)
        float y[16], mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = s[r >> 2][r & 3] * sc;
        if (!whole) kv8_masked(a.mask, pos, key0, y);
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, y[r]);
        const float ev = kv8_exponent(vsn);
        if (mmi_any(live && ref.outgrown(mx, ev))) {       // (the tile's other columns hold anything)
            float fewer, less;
            ref.move(mx, ev, [](float x) { return mmi_rows_max(x); }, fewer, less);
            l *= fewer;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= less;
        }
        const float times = ref.times(vsn, mx);
        u32x4 pf[2][NS];
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            y[r] = mmi_fast_exp2f(y[r] - ref.r);
            sum += y[r];
        }
        l += sum;
#pragma unroll
        for (int u = 0; u < 2; ++u) kv8_split8<NS>(y + 8 * u, times, pf[u]);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            u32x4 lo, hi;
            C::fragments(vw[d], lo, hi);
#pragma unroll
            for (int n = NS - 1; n >= 0; --n) {
                acc[d] = mmi_mfma_f16_16x16x32(lo, pf[0][n], acc[d]);
                acc[d] = mmi_mfma_f16_16x16x32(hi, pf[1][n], acc[d]);
            }
        }
    }
    l += mmi_shfl_xor(l, 16);
    l += mmi_shfl_xor(l, 32);
    if (kq == 0) {
        ml[0][wave][bl] = ref.r;
        ml[1][wave][bl] = ref.off;
        ml[2][wave][bl] = l;
    }
    __syncthreads();
    float R = Kv8Refs::LEAST, O = Kv8Refs::NONE, L = 0.f;
#pragma unroll
    for (int v = 0; v < WK; ++v) R = fmaxf(R, ml[0][v][bl]);
#pragma unroll
    for (int v = 0; v < WK; ++v) {
        O = fmaxf(O, ml[1][v][bl] + (ml[0][v][bl] - R));
        L += ml[2][v][bl] * mmi_fast_exp2f(ml[0][v][bl] - R);
    }
    const float f = mmi_fast_exp2f(ref.off + (ref.r - R) - O);
    const bool parts = a.few.nsplit > 1;
    const float inv = kv8_inverse(L, R, !parts && a.sink), up = mmi_fast_exp2f(O - 127.f - KV8_UP);      // (either alone is in range at the scales' ends)
    const long part = ((long)slot * a.c.kv_heads + g) * a.few.nsplit + split;
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
            v = v * inv * up;
            if (!live) continue;
            const int dim = (d0 + d) * 16 + 4 * kq, head = g * a.rep + col - tok * a.rep;
            if (parts) *reinterpret_cast<f32x4*>(a.few.po + (part * 16 + bl) * a.c.vdim + dim) = v;
            else kv8_store<Tr>(a, c.s.row0 + tok, head, dim, v);
        }
    }
    if (parts && wave == 0 && kq == 0) {
        a.few.pml[part * 32 + bl] = R;
        a.few.pml[part * 32 + 16 + bl] = L;
    }
}
// grid: slots of tiles, kv heads, splits
template <class In, class Tr, int NS, int D, bool E4M3>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void k_tlm_kv8_attn(TlmKv8Attn a) {
    MMI_SHARED __attribute__((aligned(16))) f32x4 ob[KV8_LDS];
    MMI_SHARED float ml[3][4][16];
    tlm_kv8_attn<In, Tr, NS, D, E4M3>(a, ob, ml, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
}

// 128 columns and not 256: with two tiles a wave, accumulators leave one workgroup on a CU and moves between register files (422 us instead of 227).
// A prompt of 4001 tokens, 32 heads of 128 over 8: 215 us, 610 TFLOP/s, half of what a large bf16 product reaches here; bound by the vector work between
// the products (exponentials, masks, the conversion of codes and weights).
// Many columns: four waves of 32 columns of one sequence and kv head walk the same keys, 32 at a time.  Codes become operand
// fragments on their way into LDS, once for all waves; 32 x 32 products read an operand half as often as 16 x 16 ones.  The scores of step
// i + 1 are formed beside the softmax of step i; keys lie two steps ahead of their use and values one, one barrier a step.
//   score rows: row 8 a + 4 h + i of the product is key 16 h + 4 a + i, so lane half h holds block h's 16 keys in order
//   LDS, fragments of 64 lanes: key fragment j (16 dimensions) at lane ^ (j & 7), value fragment (32 dimensions, 8 keys of each block) at
//   lane ^ 4 (lane / 32): what lets the writers, who have 16 codes of one key or dimension each, meet no bank twice
template <int NS, int D>
struct Kv8Tile {
    static constexpr int PER = KV8_MANY, KS = D / 16, DT = D / 32;
    static constexpr int KF = KS * 64, VF = DT * 2 * 64;                       // vectors per buffer
    static constexpr size_t smem() { return std::max({(size_t)2 * (KF + VF) * 16, (size_t)PER * D * NS * 2 + PER * 4 + KV8_ANGLES * 8, (size_t)KV8_LDS * 16}); }
};
template <class In, class Tr, int NS, int D, bool E4M3>
__device__ __forceinline__ void tlm_kv8_tile(const TlmKv8Attn& a, u32x4* lds, int slot, int g, int split) {
    typedef Kv8Code<E4M3> C;
    typedef Kv8Tile<NS, D> Z;
    constexpr int KS = Z::KS, DT = Z::DT, KU = D > 128 ? 2 : 1;      // units of 16 codes per thread and side
    // Two-part operands of 256 dimensions fill the registers: fewer fragments on their way, and the last k-steps' queries stay in LDS, where the angles were (with
    // all of them in registers 28 spilled)
    constexpr bool TIGHT = D * NS > 256;
    constexpr int FR = TIGHT ? 4 : 8, KR = TIGHT ? KS - 2 : KS;      // KR: k-steps whose queries are in registers
    static_assert((KS - KR) * NS * 64 * 4 * sizeof(u32x4) <= KV8_ANGLES * 8, "queries in the angles' place");
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = mmi_uniform(tid >> 6), cl = lane & 31, hi = lane >> 5;
    const Kv8Cols c(a, a.many, false, slot);
    kv8_tell(a.many, c, slot, g, split);
    const int i0 = 2 * split * a.many.pages;
    int i1 = min(2 * c.n, i0 + 2 * a.many.pages);
    if (i1 == 2 * c.n && c.n > 0 && c.page(c.n - 1) * TLM_PAGE + 32 > c.phi) --i1;      // (the last page's second half lies ahead of every column)
    if (c.c0 >= c.ncol || (i0 >= i1 && split > 0)) return;
    const int* bt = kv8_table(a.q, c.s.e);
    const int w0 = c.c0 + wave * 32;                  // the wave's first column
    const bool busy = w0 < c.ncol;
    const int plo = c.s.pos0 + min(w0, c.ncol - 1) / a.rep, phi = c.s.pos0 + min(w0 + 31, c.ncol - 1) / a.rep;
    const int col = min(w0 + cl, c.ncol - 1), tok = col / a.rep, head = g * a.rep + col - tok * a.rep;
    // ---- codes -> LDS
    u32x4 *kb = lds, *vb = lds + 2 * Z::KF;
    u32x4 kr[KU], vr[KU];
    int kput[KU], vput[KU];
    bool kon[KU], von[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
        const int n = tid + 256 * u, nk = a.c.dim / 16, key = n / nk, j = n - key * nk;
        kon[u] = key < 32;
        kput[u] = j * 64 + ((8 * ((key >> 2) & 3) + 4 * (key >> 4) + (key & 3)) ^ (j & 7));
        const int d = n >> 1, b = n & 1;
        von[u] = d < a.c.vdim;
        vput[u] = (d >> 5) * 128 + ((b * 32 + (d & 31)) ^ (4 * b));
    }
    // pages of steps: a step's place is found when its keys are asked for, and handed down to its values and scales
    struct At { long unit; int key0; bool have; };
    Kv8Pages pages;
    pages.fill(a, c, bt, i0 >> 1);
    auto find = [&](int i) __attribute__((always_inline)) {       // (past the end: the last step again)
        i = min(i, i1 - 1);
        const int p = pages.at(a, c, bt, i >> 1);
        return At{(long)max(p, 0) * a.c.kv_heads + g, c.page(i >> 1) * TLM_PAGE + 32 * (i & 1), p >= 0};
    };
    auto load_k = [&](const At& z) __attribute__((always_inline)) {
        const uint8_t* p = a.c.k + (z.unit * TLM_PAGE + (z.key0 & 32)) * a.c.dim;
#pragma unroll
        for (int u = 0; u < KU; ++u)
            if (kon[u]) kr[u] = *(const u32x4*)(p + 16 * (tid + 256 * u));
    };
    auto load_v = [&](const At& z) __attribute__((always_inline)) {
        const uint8_t* p = a.c.v + z.unit * a.c.vdim * TLM_PAGE + (z.key0 & 32);
#pragma unroll
        for (int u = 0; u < KU; ++u)
            if (von[u]) vr[u] = *(const u32x4*)(p + ((tid + 256 * u) >> 1) * TLM_PAGE + 16 * (tid & 1));
    };
    At z0, z1, z2;                                         // steps i, i + 1, i + 2
    if (i0 < i1) {
        z0 = find(i0);
        load_k(z0);
    }
    u32x4 q[KR][NS], *ql = lds + Z::PER * D * NS / 8 + Z::PER / 4 + wave * (KS - KR) * NS * 64 + lane;      // dimensions 16 s + 8 hi ..
    float back;
    {
        float* turned = reinterpret_cast<float*>(lds + Z::PER * D * NS / 8);      // inverse factors, then angles
        kv8_queries<In, NS, D>(a, c, Z::PER, g, turned + Z::PER, turned, [&](int n, int k, int p) __attribute__((always_inline)) {
            return lds + (((n >> 5) * KS + (k >> 1)) * NS + p) * 64 + 32 * (k & 1) + (n & 31);
        });
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int p = 0; p < NS; ++p) (j < KR ? q[j < KR ? j : 0][p] : ql[((j - KR) * NS + p) * 64]) = lds[((wave * KS + j) * NS + p) * 64 + lane];
        back = turned[wave * 32 + cl] * a.mask.scale;
        __syncthreads();                                   // (their memory takes keys and values)
    }
    for (int i = tid; i < 2 * Z::KF; i += 256)
        if ((i % Z::KF) / 64 >= a.c.dim / 16) kb[i] = u32x4{0u, 0u, 0u, 0u};      // (dimensions past the head's)
    auto put_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            u32x4 lo, up;
            C::fragments(kr[u], lo, up);
            if (kon[u]) {
                kb[buf * Z::KF + kput[u]] = lo;
                kb[buf * Z::KF + kput[u] + 32] = up;
            }
        }
    };
    auto put_v = [&](int buf, int key0) __attribute__((always_inline)) {
        const bool whole = kv8_whole(a.mask, c.plo, c.phi, key0, 32);
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            u32x4 lo, up;
            C::fragments(whole ? vr[u] : kv8_quiet<E4M3>(c, a.mask, key0 + 16 * (tid & 1), vr[u]), lo, up);
            if (von[u]) {
                vb[buf * Z::VF + vput[u]] = lo;
                vb[buf * Z::VF + vput[u] + 64] = up;
            }
        }
    };
    float ks = 0.f, vs = 0.f;
    auto load_s = [&](const At& z) __attribute__((always_inline)) {
        const long n = z.unit * KV8_PARTS + (z.key0 >> 4 & 2) + hi;
        ks = a.c.ks[n];
        vs = a.c.vs[n];
    };
    f32x16 acc[DT];
    Kv8Refs ref;
    float l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    f32x16 s[2];
    u32x4 fr[FR];                                          // operand fragments, asked for so many at a time
    auto scores = [&](int set, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[set][r] = 0.f;
#pragma unroll
        for (int j0 = 0; j0 < KS; j0 += FR) {
#pragma unroll
            for (int j = 0; j < FR; ++j)
                if (j0 + j < KS) fr[j] = kb[buf * Z::KF + (j0 + j) * 64 + (lane ^ ((j0 + j) & 7))];
            mmi_sched_barrier();
#pragma unroll
            for (int j = 0; j < FR; ++j)
                if (j0 + j < KS)
#pragma unroll
                    for (int n = NS - 1; n >= 0; --n)
                        s[set] = mmi_mfma_f16_32x32x16(fr[j], j0 + j < KR ? q[j0 + j < KR ? j0 + j : 0][n] : ql[((j0 + j - KR) * NS + n) * 64], s[set]);
        }
    };
    const int vl = lane ^ (4 * hi);
    auto step = [&](int i, int set) __attribute__((always_inline)) {      // scores of step i in `set`, keys of step i + 1 in LDS, of step i + 2 in registers
        const int key0 = z0.key0;
        const bool now = z0.have;
        const float ksn = ks, vsn = vs;
        load_s(z1);
        if (busy) scores(set ^ 1, set ^ 1);
        if (busy && now && key0 <= phi) {
            const bool whole = kv8_whole(a.mask, plo, phi, key0, 32);
            const float ev = kv8_exponent(vsn);
            u32x4 pf[2][NS];
            const float sc = ksn * back;
            float mx = -INFINITY, sum = 0.f, y[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] = s[set][r] * sc;
            if (!whole) kv8_masked(a.mask, c.s.pos0 + tok, key0 + 16 * hi, y);
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, y[r]);
            if (mmi_any(w0 + cl < c.ncol && ref.outgrown(mx, ev))) {       // (the tile's other columns hold anything)
                float fewer, less;
                ref.move(mx, ev, [](float x) { return mmi_halves_max(x); }, fewer, less);
                l *= fewer;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] *= less;
            }
            const float times = ref.times(vsn, mx);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                y[r] = mmi_fast_exp2f(y[r] - ref.r);
                sum += y[r];
            }
            l += sum;
#pragma unroll
            for (int u = 0; u < 2; ++u) kv8_split8<NS>(y + 8 * u, times, pf[u]);
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += FR / 2) {
#pragma unroll
                for (int k = 0; k < FR; ++k)
                    if (d0 + k / 2 < DT) fr[k] = vb[set * Z::VF + (2 * d0 + k) * 64 + vl];
                mmi_sched_barrier();
#pragma unroll
                for (int k = 0; k < FR; ++k)
                    if (d0 + k / 2 < DT)
#pragma unroll
                        for (int n = NS - 1; n >= 0; --n) acc[d0 + k / 2] = mmi_mfma_f16_32x32x16(fr[k], pf[k & 1][n], acc[d0 + k / 2]);
            }
        }
        put_k(set);
        put_v(set ^ 1, z1.key0);
        z0 = z1;
        z1 = z2;
        z2 = find(i + 3);
        load_k(z2);
        load_v(z1);
        __syncthreads();
    };
    if (i0 < i1) {                                         // (step i0 is set 0: splits hold whole pages)
        put_k(0);
        z1 = find(i0 + 1);
        load_k(z1);
        load_v(z0);
        load_s(z0);
        __syncthreads();
        if (busy) scores(0, 0);
        put_k(1);
        put_v(0, z0.key0);
        z2 = find(i0 + 2);
        load_k(z2);
        load_v(z1);
        __syncthreads();
        for (int i = i0; i < i1; i += 2) {
            step(i, 0);
            if (i + 1 < i1) step(i + 1, 1);
        }
    }
    const bool parts = a.many.nsplit > 1;
    const long part = ((long)slot * a.c.kv_heads + g) * a.many.nsplit + split;
    const int n = wave * 32 + cl;                          // column of the group
    const float L = mmi_halves_sum(l), inv = kv8_inverse(L, ref.r, !parts && a.sink), up = mmi_fast_exp2f(ref.off - 127.f - KV8_UP);
    if (c.c0 + n >= c.ncol) return;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int dim = 32 * d + 8 * r + 4 * hi;
            const f32x4 v = f32x4{acc[d][4 * r], acc[d][4 * r + 1], acc[d][4 * r + 2], acc[d][4 * r + 3]} * inv * up;
            if (dim >= a.c.vdim) continue;
            if (parts) *reinterpret_cast<f32x4*>(a.many.po + (part * Z::PER + n) * a.c.vdim + dim) = v;
            else kv8_store<Tr>(a, c.s.row0 + tok, head, dim, v);
        }
    if (parts && hi == 0) {
        a.many.pml[part * 2 * Z::PER + n] = ref.r;
        a.many.pml[part * 2 * Z::PER + Z::PER + n] = L;
    }
}
// Calls that may bring sequences of either kind: both in one launch, they share nothing.  grid: the many's kv heads x group slots (a head's groups
// on one XCD; the last groups, which see most keys, first) x splits, then the few's kv heads x slots x splits
template <class In, class Tr, int NS, int D, bool E4M3>
__global__ __launch_bounds__(256, D * NS <= 128 ? 2 : 1) void k_tlm_kv8_tile(TlmKv8Attn a, int many, int few_slots) {
    MMI_DYN_SHARED(u32x4, lds);
    MMI_SHARED float ml[3][4][16];
    const int G = a.c.kv_heads;
    int b = (int)blockIdx.x;
    if (a.rest) kv8_rest_around(a.q, b, (int)gridDim.x, [&](int row) __attribute__((always_inline)) {
        for (int g = 0; g < G; ++g) kv8_clear<Tr>(a, row, g);
    });
    if (b < many) {
        const int slots = many / (G * a.many.nsplit), split = b / (G * slots);
        b -= split * G * slots;
        tlm_kv8_tile<In, Tr, NS, D, E4M3>(a, lds, slots - 1 - b / G, b % G, split);
    } else {
        b -= many;
        tlm_kv8_attn<In, Tr, NS, D, E4M3>(a, reinterpret_cast<f32x4*>(lds), ml, b / G % few_slots, b % G, b / (G * few_slots));
    }
}

// The splits of one column -> output.  A chain of two round trips behind a launch: 3.9 us for 5 sequences (the wide one: 5.0), 5.3 us for 31 splits of
// one and 5.6 for 56 (the other: 8.6), 7.9 us for 16 sequences with 560 tokens (the wide one: 46).
//  grid: columns of all slots (first the few's, then the many's), kv heads.
// Up to 16 splits (WIDE false): a wave for every 64 / (vdim / 4) columns, four dimensions a lane, eight partial sums asked for at once.  More: a
// workgroup per column, 16 groups of lanes take every 16th split, and their sums meet in LDS.
MMI_HD int kv8_joined(int cols, int vdim, bool wide) { return wide ? cols : (cols + 256 / vdim - 1) / (256 / vdim); }      // waves (wide: workgroups) per slot
template <class Tr, bool WIDE>
__global__ __launch_bounds__(256) void k_tlm_kv8_combine(TlmKv8Attn a, int first_many, int all) {
    const int tid = (int)threadIdx.x, wave = mmi_uniform(tid >> 6), at = WIDE ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
    if (at >= all) return;
    const bool few = at < first_many;
    const Kv8Share& h = few ? a.few : a.many;
    const int b = at - (few ? 0 : first_many), each = kv8_joined(h.cols, a.c.vdim, WIDE), slot = b / each, per = h.z.per, g = (int)blockIdx.y;
    const long part = ((long)slot * a.c.kv_heads + g) * h.nsplit;
    const int cols = mmi_load_const(h.what + 4 * slot), ns = mmi_load_const(h.what + 4 * slot + 1), row0 = mmi_load_const(h.what + 4 * slot + 2), c0 = mmi_load_const(h.what + 4 * slot + 3);
    if constexpr (!WIDE) {
        const int lane = tid & 63, G = a.c.vdim / 4, at_once = 64 / G, n = (b - slot * each) * at_once + lane / G, d = 4 * (lane % G);
        const bool on = lane / G < at_once && n < h.cols;
        const float *ml0 = h.pml + part * 2 * per, *po0 = h.po + part * per * a.c.vdim;
        const unsigned at_ml = on ? n : 0, at_po = at_ml * a.c.vdim + d;
        const int step = per * a.c.vdim;                   // (a split's part: addresses are a scalar and a lane's offset)
        float m[8], l[8];
        f32x4 v[8];
        auto load = [&](int k0, int ns) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k < ns) {
                    const float* ml = ml0 + (k0 + k) * 2 * per;
                    m[k] = ml[at_ml];
                    l[k] = (ml + per)[at_ml];
                    v[k] = *(const f32x4*)(po0 + (k0 + k) * step + at_po);
                }
        };
        if (few) load(0, h.nsplit);                        // (single tokens: asked for before it is known how many splits there were)
        const int col = c0 + n;
        if (!on || n >= cols) return;
        if (!few) load(0, ns);                             // (of the slots that portions might need, half are empty)
        float R = Kv8Refs::LEAST, L = 0.f;                 // the splits so far: their reference, sum, and result (a mean: no sum of values leaves fp32)
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0;;) {
            float r = R;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k < ns) r = fmaxf(r, m[k]);
            L *= mmi_fast_exp2f(R - r);
            float all = L;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k < ns) all += l[k] *= mmi_fast_exp2f(m[k] - r);
            const float inv = kv8_inverse(all, r, k0 + 8 >= ns && a.sink);
            o *= L * inv;
            R = r;
            L = all;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k < ns) o += v[k] * (l[k] * inv);
            if ((k0 += 8) >= ns) break;
            load(k0, ns);
        }
        const int tok = col / a.rep;
        kv8_store<Tr>(a, row0 + tok, g * a.rep + col - tok * a.rep, d, o);
    } else {
        MMI_SHARED float wt[256], red[4][2];
        MMI_SHARED __attribute__((aligned(16))) f32x4 sum[256];
        const int n = b - slot * each;
        const int col = c0 + n;                            // (ns: at most 256)
        if (n >= cols) return;
        const int tok = col / a.rep, head = g * a.rep + col - tok * a.rep;
        float m = Kv8Refs::LEAST, l = 0.f;
        if (tid < ns) {
            m = h.pml[(part + tid) * 2 * per + n];
            l = h.pml[(part + tid) * 2 * per + per + n];
        }
        const float wm = mmi_wave_max_f32(m);
        if ((tid & 63) == 0) red[wave][0] = wm;
        __syncthreads();
        const float R = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
        l *= mmi_fast_exp2f(m - R);
        const float wl = mmi_wave_sum_down(l);
        if ((tid & 63) == 0) red[wave][1] = wl;
        __syncthreads();
        wt[tid] = l * kv8_inverse((red[0][1] + red[1][1]) + (red[2][1] + red[3][1]), R, a.sink);
        __syncthreads();
        const int q = tid & 15, k = tid >> 4;
        for (int d0 = 0; d0 < a.c.vdim; d0 += 64) {
            const int d = d0 + 4 * q;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (d < a.c.vdim)
#pragma unroll 4
                for (int s = k; s < ns; s += 16) v += *(const f32x4*)(h.po + ((part + s) * per + n) * a.c.vdim + d) * wt[s];
            if (d0) __syncthreads();
            sum[tid] = v;
            __syncthreads();
            if (k == 0 && d < a.c.vdim) {
#pragma unroll
                for (int i = 1; i < 16; ++i) v += sum[16 * i + q];
                kv8_store<Tr>(a, row0 + tok, head, d, v);
            }
        }
    }
}
