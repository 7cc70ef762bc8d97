// Beam search: the choice over beams and vocabulary, and the beams' states moved to where their children are.
//
//   candidate (beam k, token v) of a request: score s[k] + x[k, v] - log sum exp x[k, :], ranked by score / length^alpha
//   finished beam: one candidate, its end token at the score it has
//
// Two launches: every wave takes BEAM_CHUNK logits of a row - its maximum, its sum of exponentials, and the best `beams` of it - and a workgroup per
// request ranks what the waves found.  A row's own order is that of its logits, compared as they are; rows are compared in 64 bits.
#pragma once
#include "tlm_common.h"

constexpr int BEAM_CHUNK = 1024, BEAM_TENSORS = 48, BEAM_LISTS = 1024;
// More candidates than this: their lists' first ones are looked at before the rest (2048 candidates of one request take 10.6 us with it and 10.1 us without,
// 4096 of 16 requests 12.7 and 15.5 us, 32768 of 2 requests 35 and 216 us).
constexpr int BEAM_FIRSTS = 2048;

struct TlmBeamArgs {
    const void* x; long ld;              // logits, row stride in elements
    int V, beams, chunks;                // chunks = ceil(V / BEAM_CHUNK)
    const float* score;                  // [batch][beams]
    const int* length;                   // null: no lengths
    const uint8_t* done;                 // null: none is finished
    int eos;
    double alpha;
    float* wm; double* ws;               // [row][chunk]: maximum, sum of e^(x - maximum)
    float* wx; int* wi;                  // [row][chunk][beams]: best logits and their tokens, in order; BEAM_NONE where there are fewer
    float* out_score; int* out_parent; int* out_token; uint8_t* out_done; int* out_length;
};
constexpr int BEAM_NONE = 0x7fffffff;
// Largest length penalty.  Lengths are below 2^31, so 1 / length^alpha lies between 2^-496 and 2^496: a finite score's rank is finite, and -infinity
// stays one.  (An infinity times zero would be a NaN, before and behind nobody: fewer candidates than beams.)
constexpr float BEAM_PENALTY = 16.f;

// before in the order: the larger value, the lower index where they are equal
template <class T>
__device__ __forceinline__ bool beam_better(T x, int i, T y, int j) { return x > y || (x == y && i < j); }

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

// e^(d + low), d <= 0, as 2^(d log2 e) with the product's low part carried along: a term's error is that of two exponentials good to one unit and of
// their product's rounding, 2^-21.7 at most, however large d.  A row's sum, whose logarithm is added to scores that it puts in order, has been off by
// up to 2^-22.3 (40 960 rows of 2 to 65521 logits).
__device__ __forceinline__ float beam_exp(float d, float low) {
    constexpr float L = 1.44269504f, LL = 1.92596299e-8f;
    d = d < -200.f ? -200.f : d;                           // (zero either way; a mask's -3e38 would leave infinities)
    const float p = L * d;
    return mmi_fast_exp2f(mmi_fma(L, low, mmi_fma(LL, d, mmi_fma(L, d, -p)))) * mmi_fast_exp2f(p);
}

// A wave's best: the `beams`-th largest of the lanes' maxima is a bound that as many logits reach, and few more do, one or two beyond `beams` of
// 1024 distinct ones: these are put side by side and ranked by counting who is before whom.  Where more than 64 reach it (equal logits), they are
// taken out one at a time.  Reads the logits once: 128 rows of 65521 fp32 13 us, 2.5 TB/s, 4 rows of 32000 5.3 us.  grid: chunks / 4, rows
template <class In>
__global__ __launch_bounds__(256) void k_tlm_beam_rows(TlmBeamArgs a) {
    constexpr int N = BEAM_CHUNK / 64;                     // logits per lane, in runs of four
    MMI_SHARED float cx[4][64];
    MMI_SHARED int ci[4][64];
    const int row = (int)blockIdx.y, lane = mmi_lane(), wave = mmi_uniform((int)threadIdx.x >> 6), chunk = (int)blockIdx.x * 4 + wave, K = a.beams;
    if (chunk >= a.chunks || (a.done && a.done[row])) return;
    const In* x = (const In*)a.x + (long)row * a.ld;
    const int v0 = chunk * BEAM_CHUNK + 4 * lane;
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
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n) top = fmaxf(top, v[n]);    // (NaN is passed over here and makes the sum one)
    const float m = mmi_wave_max_f32(top);
    float s = 0.f;                                         // (places past the vocabulary's end hold -infinity)
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float e = beam_exp(v[n] - m, 0.f);
        s += v[n] == -INFINITY ? 0.f : e;
    }
    double sum = (double)s;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) sum += mmi_shfl_xor(sum, k);
    const long part = (long)row * a.chunks + chunk;
    if (lane == 0) {
        a.wm[part] = m;
        a.ws[part] = sum;
    }
    float* wx = a.wx + part * K;
    int* wi = a.wi + part * K;
    // the bound (of lanes with equal maxima each counts)
    float bound = m;
    {
        float left = top;
        for (int found = 0;;) {
            const uint64_t at = mmi_ballot(left == bound);
            found += __builtin_popcountll(at);
            if (found >= K || bound == -INFINITY) break;
            if (left == bound) left = -INFINITY;
            bound = mmi_wave_max_f32(left);
        }
    }
    int count = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const bool in = v[n] >= bound && token(n) < a.V;
        const uint64_t at = mmi_ballot(in);
        if (!at) continue;
        const int k = count + mmi_below(at);
        if (in && k < 64) {
            cx[wave][k] = v[n];
            ci[wave][k] = token(n);
        }
        count += __builtin_popcountll(at);
    }
    if (count <= 64) {
        mmi_wave_sync();
        const float y = lane < count ? cx[wave][lane] : -INFINITY;
        const int i = lane < count ? ci[wave][lane] : BEAM_NONE;
        int rank = 0;
        for (int k = 0; k < count; ++k) rank += beam_better(cx[wave][k], ci[wave][k], y, i) ? 1 : 0;
        if (lane < count && rank < K) {
            wx[rank] = y;
            wi[rank] = i;
        }
        if (lane >= count && lane < K) {
            wx[lane] = -INFINITY;
            wi[lane] = BEAM_NONE;
        }
        return;
    }
    float px = INFINITY;                                   // the one taken last
    int pi = -1;
    for (int k = 0; k < K; ++k) {
        float y = -INFINITY;
        int i = BEAM_NONE;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float z = v[n] == v[n] ? v[n] : -INFINITY;
            if (token(n) < a.V && beam_better(px, pi, z, token(n)) && beam_better(z, token(n), y, i)) y = z, i = token(n);
        }
        px = mmi_wave_max_f32(y);
        pi = (int)(0x7fffffffu - mmi_wave_max_u32(y == px ? 0x7fffffffu - (unsigned)i : 0u));
        if (lane == 0) {
            wx[k] = px;
            wi[k] = pi;
        }
    }
}

// A workgroup per request: 4096 of its candidates at a time in registers, 16 a lane, beside the best found so far.  As in the rows, a bound that
// `beams` lanes of one wave reach leaves few to be ranked by counting; ranks rounded to 32 bits keep their order, which is all a bound needs.  A
// candidate's place is beam * V + token.  Latency from end to end, chunks' sums, their logarithms,
// candidates, bound, ranks: 6.6 us for 4 beams of 32000, 11.4 us for 16 requests with 8 beams of 65521.  (Candidates taken one at a time, a maximum over the
// workgroup for each: 25 us there.)
__global__ __launch_bounds__(256) void k_tlm_beam_pick(TlmBeamArgs a) {
    constexpr int N = 16;
    MMI_SHARED double base[BEAM_MAX], inv[BEAM_MAX], bx[2][4], kx[2][BEAM_MAX];      // base: score - log sum exp; inv: 1 / length^alpha; kx: the best, in order
    MMI_SHARED int kind[BEAM_MAX], bi[2][4], kp[2][BEAM_MAX];                        // kind 0: a row of logits; 1: finished; 2: no candidate with a chance
    MMI_SHARED float ks[2][BEAM_MAX], wb[4], cs[4][64];
    MMI_SHARED double cx[4][64];
    MMI_SHARED int cp[4][64], cn[4], pick[BEAM_LISTS];
    const int b = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.beams;
    // candidate n of the request: entry n % K of chunk n / K % chunks of beam n / K / chunks
    const unsigned per = (unsigned)a.chunks * (unsigned)K;
    const int all = K * (int)per;
    const long first = (long)b * all;
    double x[N + 1];
    int p[N + 1];
    float y[N + 1];
    int total = all;                                       // candidates that are looked at
    bool some = false;                                     // they are those of the lists in pick
    const float one_k = 1.f / (float)K, one_per = 1.f / (float)per;
    auto quotient = [](int n, int d, float one) __attribute__((always_inline)) {      // n / d (n is below 2^21: at most one off)
        int k = (int)((float)n * one);
        if (k * d > n) --k;
        else if ((k + 1) * d <= n) ++k;
        return k;
    };
    auto place = [&](int n) __attribute__((always_inline)) {
        if (!some) return n;
        const int l = quotient(n, K, one_k);
        return pick[l] * K + n - l * K;
    };
    auto ask = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (j && n0 + 256 * j >= total) break;
            const int n = place(min(n0 + tid + 256 * j, total - 1));
            p[j] = a.wi[first + n];
            y[j] = a.wx[first + n];
        }
    };
    // the largest value that `beams` lanes of the wave reach (-infinity: there is none)
    auto reached = [&](float top) __attribute__((always_inline)) {
        float bound = mmi_wave_max_f32(top), left = top;
        for (int found = 0;;) {
            found += __builtin_popcountll(mmi_ballot(left == bound));
            if (found >= K || bound == -INFINITY) break;
            if (left == bound) left = -INFINITY;
            bound = mmi_wave_max_f32(left);
        }
        return bound;
    };
    if (all <= BEAM_FIRSTS) ask(0);
    // two rows a wave at once, a chunk a lane; then a beam a lane: its score and its length's power, in 64 bits
    const bool mine = tid < K, done = mine && a.done && a.done[b * K + tid];
    const double score = mine ? (double)a.score[b * K + tid] : 0.;
    const int len = mine && a.length ? a.length[b * K + tid] + (done ? 0 : 1) : 1;
    for (int k = wave; k < K; k += 8) {
        const long r0 = (long)(b * K + k) * a.chunks, r1 = (long)(b * K + min(k + 4, K - 1)) * a.chunks;
        const int at = min(lane, a.chunks - 1);
        const bool in = lane < a.chunks;
        const float m0 = a.wm[r0 + at], m1 = a.wm[r1 + at];
        const double w0 = a.ws[r0 + at], w1 = a.ws[r1 + at];
        auto sum = [&](int k, long row, float m, double w) __attribute__((always_inline)) {
            float M = in ? m : -INFINITY;
            for (int i = lane + 64; i < a.chunks; i += 64) M = fmaxf(M, a.wm[row + i]);
            M = mmi_wave_max_f32(M);
            auto share = [&](float m, double w) __attribute__((always_inline)) {
                const double d = (double)m - (double)M;
                const float high = (float)d;
                return w == 0. ? 0. : w * (double)beam_exp(high, (float)(d - (double)high));
            };
            double S = in ? share(m, w) : 0.;
            for (int i = lane + 64; i < a.chunks; i += 64) S += share(a.wm[row + i], a.ws[row + i]);
#pragma unroll
            for (int i = 1; i < 64; i <<= 1) S += mmi_shfl_xor(S, i);
            if (lane == 0) {
                base[k] = (double)M;
                inv[k] = S;
            }
        };
        sum(k, r0, m0, w0);
        if (k + 4 < K) sum(k + 4, r1, m1, w1);
    }
    __syncthreads();
    if (mine) {
        const double z = done ? score : score - (base[tid] + log(inv[tid]));
        base[tid] = z;
        inv[tid] = a.alpha == 0. ? 1. : (a.alpha == 1. ? 1. / (double)max(len, 1) : pow((double)max(len, 1), -a.alpha));
        kind[tid] = z > -INFINITY && z < INFINITY ? (done ? 1 : 0) : 2;
    }
    float least = -INFINITY;                               // as many candidates as there are beams reach it
    if (all > BEAM_FIRSTS) {
        // Lists are in order, so the first ones of each tell which lists can have a candidate at all: those whose first reaches a bound that as many
        // firsts reach.
        const int lists = K * a.chunks;
        const float one_chunk = 1.f / (float)a.chunks;
        auto head = [&](int i) __attribute__((always_inline)) {
            const int k = quotient(i, a.chunks, one_chunk);
            double s = -INFINITY;
            if (kind[k] == 0) s = base[k] + (double)a.wx[first + (long)i * K];
            else if (kind[k] == 1 && i == k * a.chunks) s = base[k];
            return (float)(s * inv[k]);
        };
        __syncthreads();
        float top = -INFINITY;
#pragma unroll 4
        for (int i = tid; i < lists; i += 256) top = fmaxf(top, head(i));
        const float bound = reached(top);
        if (lane == 0) wb[wave] = bound;
        __syncthreads();
        least = fmaxf(fmaxf(wb[0], wb[1]), fmaxf(wb[2], wb[3]));
        if (least > -INFINITY) {
            int count = 0;
            for (int i0 = 0; i0 < lists; i0 += 256) count += __builtin_popcountll(mmi_ballot(i0 + tid < lists && head(min(i0 + tid, lists - 1)) >= least));
            if (lane == 0) cn[wave] = count;
            __syncthreads();
            if (cn[0] + cn[1] + cn[2] + cn[3] <= BEAM_LISTS) {
                int at = 0;
                for (int w = 0; w < wave; ++w) at += cn[w];
                for (int i0 = 0; i0 < lists; i0 += 256) {
                    const bool in = i0 + tid < lists && head(min(i0 + tid, lists - 1)) >= least;
                    const uint64_t who = mmi_ballot(in);
                    if (in) pick[at + mmi_below(who)] = i0 + tid;
                    at += __builtin_popcountll(who);
                }
                some = true;
                total = (cn[0] + cn[1] + cn[2] + cn[3]) * K;
            }
            __syncthreads();
        }
        ask(0);
    }
    x[N] = -INFINITY;
    p[N] = BEAM_NONE;
    y[N] = -INFINITY;
    int set = 0;
    for (int n0 = 0; n0 < total; n0 += 256 * N, set ^= 1) {
        if (n0) ask(n0);
        __syncthreads();
        if (n0 && tid < K) {                               // (place BEAM_NONE: there was none)
            x[N] = kx[set ^ 1][tid];
            p[N] = kp[set ^ 1][tid];
            y[N] = ks[set ^ 1][tid];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (n0 + 256 * j >= total) {                   // (one request's few candidates leave most places empty)
                p[j] = BEAM_NONE;
                continue;
            }
            const bool there = n0 + tid + 256 * j < total;
            const int n = place(min(n0 + tid + 256 * j, total - 1));
            int k = quotient(n, (int)per, one_per);
            k = min(k, K - 1);
            const int h = n - k * (int)per;
            int token = there ? p[j] : BEAM_NONE;
            double s = -INFINITY;
            if (kind[k] == 0) {
                if (token != BEAM_NONE) s = base[k] + (double)y[j];
            } else {                                       // no logits to choose from: the end token, then what else there is, in order, as the first entries
                token = kind[k] == 2 ? h : (h == 0 ? a.eos : (h - 1 < a.eos ? h - 1 : h));
                if (h >= K || !there || token >= a.V) token = BEAM_NONE;
                if (kind[k] == 1 && h == 0) s = base[k];
            }
            x[j] = s * inv[k];
            y[j] = (float)s;
            p[j] = token == BEAM_NONE ? BEAM_NONE : k * a.V + token;      // (below 2^25)
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j <= N; ++j)
            if (j == N || n0 + 256 * j < total) top = fmaxf(top, p[j] == BEAM_NONE ? -INFINITY : (float)x[j]);
        float bound = reached(top);
        if (lane == 0) wb[wave] = bound;
        __syncthreads();
        bound = fmaxf(fmaxf(fmaxf(wb[0], wb[1]), fmaxf(wb[2], wb[3])), least);
        int count = 0;
#pragma unroll
        for (int j = 0; j <= N; ++j) {
            if (j < N && n0 + 256 * j >= total) continue;
            const bool in = p[j] != BEAM_NONE && (float)x[j] >= bound;
            const uint64_t at = mmi_ballot(in);
            if (!at) continue;
            const int k = count + mmi_below(at);
            if (in && k < 64) {
                cx[wave][k] = x[j];
                cp[wave][k] = p[j];
                cs[wave][k] = y[j];
            }
            count += __builtin_popcountll(at);
        }
        if (lane == 0) cn[wave] = count;
        if (tid < K) kp[set][tid] = BEAM_NONE;             // (fewer candidates than beams so far)
        __syncthreads();
        if (max(max(cn[0], cn[1]), max(cn[2], cn[3])) <= 64) {
            if (lane < count) {
                const double m = cx[wave][lane];
                const int q = cp[wave][lane];
                int rank = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    for (int k = 0; k < cn[w]; ++k) rank += beam_better(cx[w][k], cp[w][k], m, q) ? 1 : 0;
                if (rank < K) {
                    kx[set][rank] = m;
                    kp[set][rank] = q;
                    ks[set][rank] = cs[wave][lane];
                }
            }
            continue;
        }
        // many candidates of equal rank: one at a time
        for (int n = 0; n < K; ++n) {
            double m = -INFINITY;
            int q = BEAM_NONE;
            float s = -INFINITY;
#pragma unroll
            for (int j = 0; j <= N; ++j)
                if (p[j] != BEAM_NONE && beam_better(x[j], p[j], m, q)) m = x[j], q = p[j], s = y[j];
            const int mine = q;
            double least = -m;
            mmi_wave_pair_min(least, q);
            if (lane == 0) {
                bx[n & 1][wave] = least;
                bi[n & 1][wave] = q;
            }
            __syncthreads();
            least = bx[n & 1][0];
            q = bi[n & 1][0];
#pragma unroll
            for (int w = 1; w < 4; ++w) mmi_pair_min(least, q, bx[n & 1][w], bi[n & 1][w]);
            if (mine == q && q != BEAM_NONE) {             // (places differ: one lane's)
                kx[set][n] = -least;
                kp[set][n] = q;
                ks[set][n] = s;
#pragma unroll
                for (int j = 0; j <= N; ++j) p[j] = p[j] == q ? BEAM_NONE : p[j];
            }
        }
    }
    __syncthreads();
    set ^= 1;
    if (tid < K) {
        const int o = b * K + tid, k = kp[set][tid] / a.V, t = kp[set][tid] - k * a.V, row = b * K + k;
        const bool done = a.done && a.done[row];
        a.out_score[o] = ks[set][tid];
        a.out_parent[o] = k;
        a.out_token[o] = t;
        if (a.out_done) a.out_done[o] = done || t == a.eos;
        if (a.out_length) a.out_length[o] = (a.length ? a.length[row] : 0) + (done ? 0 : 1);
    }
}

// ---- reorder: row r of a request's `beams` rows becomes a copy of what row parent[r] was, in place ------------------------------
struct TlmReorder {
    struct T { char* p; long stride; unsigned units, block0; int unit; } t[BEAM_TENSORS];      // base, bytes from row to row, units per row and their bytes, first workgroup
    int n, beams;
    const int* parent;                   // [requests][beams], within the request
    const int* row;                      // null: rows in order
};
// A lane owns a unit of the request's rows: it has read all of it before it writes any, so rows may change places.  Rows that stay are not written,
// and in their place a row that some other one needs is asked for again: a load behind a branch would wait for the one before it (315 us
// instead of 188 for 64 rows of 13 MB, of which random parents have 30 read and 43 written: 0.98 GB at 5.3 TB/s, a copy of 1 GiB 5.2; a row that
// two children take is read once).  Four rows of 3.4 MB: 5.5 us, a launch and one round trip.  Instances by the beams, since their registers are a lane's.
template <class U, int K>
__device__ __forceinline__ void beam_move(const TlmReorder::T& t, const int (&from)[K], const int (&to)[K], unsigned moved, unsigned u) {
    U v[K];
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = ((const U*)(t.p + (long)from[i] * t.stride))[u];
    mmi_sched_barrier();
#pragma unroll
    for (int i = 0; i < K; ++i)
        if (moved >> i & 1) ((U*)(t.p + (long)to[i] * t.stride))[u] = v[i];
}
// grid: blocks of units of all tensors, requests
template <int K>
__global__ __launch_bounds__(256) void k_tlm_reorder(TlmReorder a) {
    const int base = (int)blockIdx.y * a.beams;
    int from[K], to[K], some = -1;
    unsigned moved = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        to[i] = min(i, a.beams - 1);
        from[i] = mmi_load_const(a.parent + base + to[i]);
        if (i < a.beams && from[i] != i && from[i] >= 0 && from[i] < a.beams) {      // (a parent that does not exist: the row stays)
            moved |= 1u << i;
            some = from[i];
        }
    }
    if (!moved) return;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int f = base + (moved >> i & 1 ? from[i] : some), r = base + to[i];
        from[i] = a.row ? mmi_load_const(a.row + f) : f;
        to[i] = a.row ? mmi_load_const(a.row + r) : r;
    }
    int n = 0;
    while (n + 1 < a.n && a.t[n + 1].block0 <= blockIdx.x) ++n;
    const TlmReorder::T t = a.t[n];
    const unsigned u = (blockIdx.x - t.block0) * 256u + threadIdx.x;
    if (u >= t.units) return;
    if (t.unit == 16) beam_move<u32x4, K>(t, from, to, moved, u);
    else if (t.unit == 4) beam_move<uint32_t, K>(t, from, to, moved, u);
    else beam_move<uint8_t, K>(t, from, to, moved, u);
}
