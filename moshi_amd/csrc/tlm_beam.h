// Beam search: the choice over beams and vocabulary, and the beams' states moved to where their children are.
//
//   candidate (beam k, token v) of a request: score s[k] + x[k, v] - log sum exp x[k, :], ranked by score / length^alpha
//   finished beam: one candidate, its end token at the score it has
//
// Two launches: every workgroup takes BEAM_CHUNK logits of a row - its maximum, its sum of exponentials, and the best BEAMS of it in order - and one
// wave per request merges these lists.  A row's own order is that of its logits, compared as they are; rows are compared in 64 bits.
#pragma once
#include "tlm_common.h"

constexpr int BEAM_MAX = 32, BEAM_CHUNK = 4096, BEAM_TENSORS = 48;

struct TlmBeamArgs {
    const void* x; long ld;              // logits, row stride in elements
    int V, beams, splits;                // splits = ceil(V / BEAM_CHUNK)
    const float* score;                  // [batch][beams]
    const int* length;                   // null: no lengths
    const uint8_t* done;                 // null: none is finished
    int eos;
    double alpha;
    float* wm; double* ws;               // [row][split]: maximum, sum of e^(x - maximum)
    float* wx; int* wi;                  // [row][split][beams]: best logits and their tokens
    float* out_score; int* out_parent; int* out_token; uint8_t* out_done; int* out_length;
};

// the larger of two (value, index) pairs, the lower index where the values are equal
template <class T>
__device__ __forceinline__ bool beam_better(T x, int i, T y, int j) { return x > y || (x == y && i < j); }
template <class T>
__device__ __forceinline__ void beam_wave_best(T& x, int& i) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const T ox = mmi_shfl_xor(x, m);
        const int oi = mmi_shfl_xor(i, m);
        const bool take = beam_better(ox, oi, x, i);
        x = take ? ox : x;
        i = take ? oi : i;
    }
}

typedef f32x4 f32x4_loose __attribute__((aligned(4)));       // (rows of odd lengths begin anywhere)
typedef u32x2 u32x2_loose __attribute__((aligned(2)));
__device__ __forceinline__ f32x4 beam_load4(const float* p) { return *(const f32x4_loose*)p; }
__device__ __forceinline__ f32x4 beam_load4(const uint16_t* p) {
    const u32x2 w = *(const u32x2_loose*)p;
    return f32x4{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16),
                 __builtin_bit_cast(float, w[1] & 0xffff0000u)};
}
__device__ __forceinline__ float beam_load(const float* p) { return *p; }
__device__ __forceinline__ float beam_load(const uint16_t* p) { return mmi_bf16_to_f32(*p); }

// grid: chunks, rows
template <class In>
__global__ __launch_bounds__(256) void k_tlm_beam_rows(TlmBeamArgs a) {
    constexpr int N = BEAM_CHUNK / 256;                    // logits per lane, in runs of four
    MMI_SHARED float lm[4], lx[4][BEAM_MAX];
    MMI_SHARED double ls[4];
    MMI_SHARED int li[4][BEAM_MAX];
    const int row = (int)blockIdx.y, split = (int)blockIdx.x, lane = mmi_lane(), wave = mmi_uniform((int)threadIdx.x >> 6);
    if (a.done && a.done[row]) return;
    const In* x = (const In*)a.x + (long)row * a.ld;
    const int v0 = split * BEAM_CHUNK + wave * (BEAM_CHUNK / 4) + 4 * lane;
    float v[N];
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        const int at = v0 + 256 * j;
        if (at + 4 <= a.V) {
            const f32x4 w = beam_load4(x + at);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * j + r] = w[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * j + r] = at + r < a.V ? beam_load(x + at + r) : -INFINITY;
        }
    }
    auto token = [&](int n) __attribute__((always_inline)) { return v0 + 256 * (n >> 2) + (n & 3); };
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n) m = fmaxf(m, v[n]);        // (NaN is passed over here and makes the sum one)
    m = mmi_wave_max_f32(m);
    // e^d as 2^(d log2 e) with the product's low part carried along: the sum's relative error stays near 2^-28, where its logarithm is added to
    // scores whose order it decides.  Places past the vocabulary's end hold -infinity.
    constexpr float L = 1.44269504f, LL = 1.92596299e-8f;
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float d = v[n] - m;
        d = d < -200.f ? -200.f : d;                       // (zero either way; a mask's -3e38 would leave infinities)
        const float p = L * d, e = mmi_fast_exp2f(mmi_fma(LL, d, mmi_fma(L, d, -p))) * mmi_fast_exp2f(p);
        s += v[n] == -INFINITY ? 0.f : e;
    }
    double sum = (double)s;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) sum += mmi_shfl_xor(sum, k);
    // the wave's best, one at a time: every lane keeps its best one, and looks through the rest when that is taken
    float best;
    int at;
    auto look = [&](float below, int after) __attribute__((always_inline)) {      // the best behind (below, after) in the order
        best = -INFINITY;
        at = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float y = v[n] == v[n] ? v[n] : -INFINITY;
            const int i = token(n);
            const bool left = i < a.V && beam_better(below, after, y, i);
            if (left && beam_better(y, i, best, at)) best = y, at = i;
        }
    };
    look(INFINITY, -1);
    for (int k = 0; k < a.beams; ++k) {
        float y = best;
        int i = at;
        beam_wave_best(y, i);
        if (lane == 0) lx[wave][k] = y, li[wave][k] = i;
        if (at == i && i != 0x7fffffff) look(y, i);
    }
    if (lane == 0) lm[wave] = m, ls[wave] = sum;
    __syncthreads();
    if (wave) return;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, lm[w]);
    const long part = (long)row * a.splits + split;
    if (lane == 0) {
        double S = 0.;
#pragma unroll
        for (int w = 0; w < 4; ++w) S += ls[w] == 0. ? 0. : ls[w] * exp((double)lm[w] - (double)M);
        a.wm[part] = M;
        a.ws[part] = S;
    }
    // the four waves' lists: 16 lanes a wave, two entries each
    float y[2];
    int i[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = (lane & 15) + 16 * h;
        y[h] = k < a.beams ? lx[lane >> 4][k] : -INFINITY;
        i[h] = k < a.beams ? li[lane >> 4][k] : 0x7fffffff;
    }
    for (int k = 0; k < a.beams; ++k) {
        const bool second = beam_better(y[1], i[1], y[0], i[0]);
        float b = second ? y[1] : y[0];
        int j = second ? i[1] : i[0];
        beam_wave_best(b, j);
        if (lane == 0) a.wx[part * a.beams + k] = b, a.wi[part * a.beams + k] = j;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (i[h] == j) y[h] = -INFINITY, i[h] = 0x7fffffff;
    }
}

// One wave per request.  A list is a row's split, in order; a lane looks after every 64th and keeps the best head among them.
__global__ __launch_bounds__(64) void k_tlm_beam_pick(TlmBeamArgs a) {
    MMI_DYN_SHARED(int, head);                             // [beams * splits]: entries of a list that are taken
    MMI_SHARED double base[BEAM_MAX], div[BEAM_MAX];       // score - log sum exp, length^alpha
    MMI_SHARED int kind[BEAM_MAX];                         // 0: a row of logits; 1: finished; 2: no candidate with a chance
    const int b = (int)blockIdx.x, lane = mmi_lane(), K = a.beams;
    if (lane < K) {
        const int row = b * K + lane;
        const bool done = a.done && a.done[row];
        const int len = a.length ? a.length[row] + (done ? 0 : 1) : 1;
        const double s = (double)a.score[row];
        double z = s;
        if (!done) {
            float M = -INFINITY;
            for (int i = 0; i < a.splits; ++i) M = fmaxf(M, a.wm[(long)row * a.splits + i]);
            double S = 0.;
            for (int i = 0; i < a.splits; ++i) {
                const double w = a.ws[(long)row * a.splits + i];
                S += w == 0. ? 0. : w * exp((double)a.wm[(long)row * a.splits + i] - (double)M);
            }
            z = s - ((double)M + log(S));
        }
        base[lane] = z;
        div[lane] = a.alpha == 0. ? 1. : pow((double)max(len, 1), a.alpha);
        kind[lane] = z > -INFINITY && z < INFINITY ? (done ? 1 : 0) : 2;
    }
    const int lists = K * a.splits;
    for (int i = lane; i < lists; i += 64) head[i] = 0;
    __syncthreads();
    // entry h of list i: its rank, and its place beam * V + token (as 64 bits: 32 beams of a vocabulary above 2^26)
    auto entry = [&](int i, int h, double& rank, double& score, int& token) __attribute__((always_inline)) {
        const int k = i / a.splits, split = i - k * a.splits;
        token = 0x7fffffff;
        score = rank = -INFINITY;
        if (h >= K) return;
        if (kind[k] != 0) {                                // a list in the first split alone: the end token, and what else there is, in order
            if (split) return;
            const int skip = kind[k] == 1 ? a.eos : a.V;
            token = kind[k] == 1 ? (h == 0 ? skip : (h - 1 < skip ? h - 1 : h)) : h;
            if (token >= a.V) token = 0x7fffffff;
            if (kind[k] == 1 && h == 0) score = base[k];
        } else {
            const long at = ((long)(b * K + k) * a.splits + split) * K + h;
            token = a.wi[at];
            score = token == 0x7fffffff ? -INFINITY : base[k] + (double)a.wx[at];
        }
        rank = score / div[k];
    };
    double best, bscore;
    int blist, btoken;
    auto look = [&]() __attribute__((always_inline)) {
        best = bscore = -INFINITY;
        blist = btoken = 0x7fffffff;
        for (int i = lane; i < lists; i += 64) {
            double r, s;
            int t;
            entry(i, head[i], r, s, t);
            // equal ranks: the lower beam, then the lower token; lists of one lane come in the order of their beams
            const bool same = blist != 0x7fffffff && i / a.splits == blist / a.splits;
            if (t != 0x7fffffff && (blist == 0x7fffffff || r > best || (r == best && same && t < btoken))) best = r, bscore = s, blist = i, btoken = t;
        }
    };
    look();
    for (int n = 0; n < K; ++n) {
        double r = best;
        int k = blist == 0x7fffffff ? 0x7fffffff : blist / a.splits, t = btoken;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double ro = mmi_shfl_xor(r, m);
            const int ko = mmi_shfl_xor(k, m), to = mmi_shfl_xor(t, m);
            const bool take = ko != 0x7fffffff && (k == 0x7fffffff || ro > r || (ro == r && (ko < k || (ko == k && to < t))));
            r = take ? ro : r;
            k = take ? ko : k;
            t = take ? to : t;
        }
        if (blist != 0x7fffffff && blist / a.splits == k && btoken == t) {      // one lane's
            const int o = b * K + n, row = b * K + k;
            const bool done = a.done && a.done[row];
            a.out_score[o] = (float)bscore;
            a.out_parent[o] = k;
            a.out_token[o] = t;
            if (a.out_done) a.out_done[o] = done || t == a.eos;
            if (a.out_length) a.out_length[o] = (a.length ? a.length[row] : 0) + (done ? 0 : 1);
            ++head[blist];
            look();
        }
    }
}

// ---- reorder: row r of a request's `beams` rows becomes a copy of what row parent[r] was, in place ------------------------------
struct TlmReorder {
    struct T { char* p; long stride; unsigned units, block0; } t[BEAM_TENSORS];      // base, bytes from row to row, units per row, first workgroup
    int n, beams;
    const int* parent;                   // [requests][beams], within the request
    const int* row;                      // null: rows in order
};
// U bytes a unit.  A lane owns a column of a request: it has read all of it before it writes any, so rows may change places.
// grid: column blocks of all tensors, requests
template <class U, int K>
__global__ __launch_bounds__(256) void k_tlm_reorder(TlmReorder a) {
    int n = 0;
    while (n + 1 < a.n && a.t[n + 1].block0 <= blockIdx.x) ++n;
    const TlmReorder::T t = a.t[n];
    const unsigned u = (blockIdx.x - t.block0) * 256u + threadIdx.x;
    if (u >= t.units) return;
    const int base = (int)blockIdx.y * a.beams;
    U v[K];
    int p[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        p[i] = i < a.beams ? a.parent[base + i] : i;
        if (p[i] < 0 || p[i] >= a.beams) p[i] = i;         // (a parent that does not exist: the row stays)
    }
    auto at = [&](int i) __attribute__((always_inline)) { return (U*)(t.p + (long)(a.row ? a.row[base + i] : base + i) * t.stride) + u; };
#pragma unroll
    for (int i = 0; i < K; ++i)
        if (p[i] != i) v[i] = *at(p[i]);
#pragma unroll
    for (int i = 0; i < K; ++i)
        if (p[i] != i) *at(i) = v[i];
}
