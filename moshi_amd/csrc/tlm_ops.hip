// Operators of the token language models behind the C ABI of include/moshi_tlm.h: the 8-bit key/value cache and its attention, beam search's
// choice and the reordering of its states.
#include "../../include/moshi_tlm.h"
#include "tlm_ops.h"
#include "tlm_beam.h"

namespace {

// Workgroups that a split of the pages aims at.  Few columns: one per CU (128, 256, 512, 1024 of them: 100 003 keys of 8 heads of 128 62, 44, 47, 59 us, of 4 heads of 256 72, 55, 73,
// 91, 64 sequences of 800 to 4096 keys 77, 77, 77, 86, eight of 8000 27, 21, 23, 30, 24 of 1500 20, 24, 25, 28); more are more parts to join.
constexpr long KV8_WORKGROUPS = 256;
// The same of k_tlm_kv8_tile (256, 384, 512: 16 sequences with 560 tokens 43, 41, 45 us, 24 with 540 tokens of 64 dimensions 53, 44, 43, a prompt of 1200 on one kv head 35, 34, 37, one
// of 100 behind 900 keys 30, 30, 36, 1260 tokens behind 2000 80, 73, 64), and where heads above 128 leave a CU one workgroup (192, 256, 384, 512: 720 tokens of 256 dimensions
// behind 1500 keys 65, 59, 91, 88).
constexpr long KV8_TILES = 384, KV8_TILES_WIDE = 256;
constexpr int KV8_MAX_SPLIT = 256;       // (k_tlm_kv8_combine: a lane each)

int check_cache(const mmi_kv_cache* c, TlmKv8Cache* out, const char* at) {
    auto bad = [&](int code, const char* what) { return mmi_fail(code, std::string(at) + ": " + what); };
    if (!c) return bad(MMI_ERR_INVALID, "null cache");
    if (c->pages < 1 || c->pages > 0x7fffffff) return bad(MMI_ERR_SHAPE, "the cache needs between 1 and 2^31 - 1 pages");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return bad(MMI_ERR_INVALID, "null cache");
    if (c->kv_heads < 1 || c->kv_heads > 65535) return bad(MMI_ERR_SHAPE, "key/value heads");
    if (c->dim < 16 || c->dim > 256 || c->dim % 16 || c->vdim < 16 || c->vdim > 256 || c->vdim % 16)
        return bad(MMI_ERR_UNSUPPORTED, "head sizes are multiples of 16 up to 256");
    if (c->codes != MMI_I8 && c->codes != MMI_F8E4M3) return bad(MMI_ERR_UNSUPPORTED, "codes are int8 or e4m3");
    if (c->rot_dim < 0 || c->rot_dim > c->dim || c->rot_dim % 8 || (c->rot_dim && !c->rot_freq)) return bad(MMI_ERR_INVALID, "rotated dimensions are a multiple of 8 up to the head size, with frequencies");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return bad(MMI_ERR_INVALID, "codes must be aligned to 16 bytes");
    *out = TlmKv8Cache{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, (int)c->pages, c->kv_heads, c->dim, c->vdim, c->codes == MMI_F8E4M3, c->rot_dim, c->rot_halves, c->rot_freq};
    return MMI_OK;
}
int check_seqs(const mmi_kv_seqs* q, TlmKv8Seqs* out, const char* at) {
    auto bad = [&](int code, const char* what) { return mmi_fail(code, std::string(at) + ": " + what); };
    if (!q || q->n < 0 || q->rows < 0) return bad(MMI_ERR_INVALID, "bad sequences");
    if (q->n && (!q->position || !q->table || q->table_ld < 1)) return bad(MMI_ERR_INVALID, "sequences need positions and a page table");
    if (!q->row0 && q->rows != q->n) return bad(MMI_ERR_SHAPE, "without row starts every sequence brings one row");
    if (q->n > 1 << 20 || q->rows > 1 << 24) return bad(MMI_ERR_SHAPE, "at most 2^20 sequences and 2^24 rows");
    *out = TlmKv8Seqs{q->n, q->rows, q->row0, nullptr, q->position, nullptr, TlmPages{q->table, q->table_ld, q->table_ld}, 0};
    return MMI_OK;
}
int check_rows(const void* p, int64_t row, int64_t head, int dtype, const char* at) {
    if (!p) return mmi_fail(MMI_ERR_INVALID, std::string(at) + ": null tensor");
    if (row < 0 || head < 0) return mmi_fail(MMI_ERR_INVALID, std::string(at) + ": negative stride");
    if (dtype != MMI_BF16 && dtype != MMI_F32) return mmi_fail(MMI_ERR_UNSUPPORTED, std::string(at) + ": bf16 or fp32");
    return MMI_OK;
}
// do the heads of rows (n elements each) lie apart, heads within rows or rows within heads?
bool rows_apart(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t n) {
    auto fits = [n](int64_t few, int64_t narrow, int64_t many, int64_t wide) { return (few == 1 || narrow >= n) && (many == 1 || (__int128)wide >= (__int128)(few - 1) * narrow + n); };
    return fits(heads, head, rows, row) || fits(rows, row, heads, head);
}
// can four elements be loaded at once?
bool aligned4(const void* p, int64_t row, int64_t head, int dtype) { return (uintptr_t)p % (dtype == MMI_F32 ? 16 : 8) == 0 && row % 4 == 0 && head % 4 == 0; }

template <class F>
int by_codes(int e4m3, F f) { return e4m3 ? f(std::true_type()) : f(std::false_type()); }

int launch_read(hipStream_t s, const TlmKv8Read& a, int dtype) {
    const long slots = kv8_slots(a.q, a.z);
    return by_codes(a.c.e4m3, [&](auto e) {
        if (dtype == MMI_F32) MMI_LAUNCH((k_tlm_kv8_read<float, decltype(e)::value>), dim3((unsigned)slots, a.c.kv_heads, 2), 64, 0, s, a);
        else MMI_LAUNCH((k_tlm_kv8_read<uint16_t, decltype(e)::value>), dim3((unsigned)slots, a.c.kv_heads, 2), 64, 0, s, a);
        MMI_CHECK_LAUNCH();
        return (int)MMI_OK;
    });
}

template <class In, class Tr, int NS, int D, bool E4M3>
int launch_attn(hipStream_t s, const TlmKv8Attn& a) {
    if (a.both) {
        constexpr size_t smem = Kv8Tile<NS, D>::smem();
        static_assert(smem <= 160 * 1024, "LDS of a CU");
        if (smem > 64 * 1024) {
            static std::atomic<uint64_t> asked{0};
            if (const int rc = mmi_allow_lds(reinterpret_cast<const void*>(&k_tlm_kv8_tile<In, Tr, NS, D, E4M3>), (int)smem, asked)) return rc;
        }
        const int slots = (int)kv8_slots(a.q, a.few.z), many = (int)kv8_slots(a.q, a.many.z) * a.c.kv_heads * a.many.nsplit;
        MMI_LAUNCH((k_tlm_kv8_tile<In, Tr, NS, D, E4M3>), (unsigned)many + (unsigned)slots * a.c.kv_heads * a.few.nsplit, 256, smem, s, a, many, slots);
    } else {
        MMI_LAUNCH((k_tlm_kv8_attn<In, Tr, NS, D, E4M3>), dim3((unsigned)kv8_slots(a.q, a.few.z), a.c.kv_heads, a.few.nsplit), 256, 0, s, a);
    }
    const bool wide = std::max(a.few.nsplit, a.both ? a.many.nsplit : 1) > 16;      // (both sides measured: k_tlm_kv8_combine)
    auto joined = [&](const Kv8Share& h) { return h.nsplit > 1 ? (int)kv8_slots(a.q, h.z) * kv8_joined(h.cols, a.c.vdim, wide) : 0; };
    const int few = joined(a.few), all = few + (a.both ? joined(a.many) : 0);
    if (all && wide) MMI_LAUNCH((k_tlm_kv8_combine<Tr, true>), dim3(all, a.c.kv_heads), 256, 0, s, a, few, all);
    else if (all) MMI_LAUNCH((k_tlm_kv8_combine<Tr, false>), dim3(mmi_cdiv(all, 4), a.c.kv_heads), 256, 0, s, a, few, all);
    MMI_CHECK_LAUNCH();
    return MMI_OK;
}
template <class In, class Tr, int NS, int D>
int launch_attn_c(hipStream_t s, const TlmKv8Attn& a) { return a.c.e4m3 ? launch_attn<In, Tr, NS, D, true>(s, a) : launch_attn<In, Tr, NS, D, false>(s, a); }
int attn_bound(const TlmKv8Cache& c) {                 // the kernels' bound on both head sizes
    const int d = std::max(c.dim, c.vdim);
    return d <= 64 ? 64 : (d <= 128 ? 128 : 256);
}
template <class In, class Tr, int NS>
int launch_attn_d(hipStream_t s, const TlmKv8Attn& a) {
    const int d = attn_bound(a.c);
    return d == 64 ? launch_attn_c<In, Tr, NS, 64>(s, a) : (d == 128 ? launch_attn_c<In, Tr, NS, 128>(s, a) : launch_attn_c<In, Tr, NS, 256>(s, a));
}
// how a kernel's `groups` (the ones that are likely to have columns) share the pages out; floats of workspace, at most `room`
size_t split_pages(const TlmKv8Attn& a, Kv8Share& h, long groups, long cap, size_t room, long aim, long step) {
    if (a.mask.window > 0)                             // positions plo - window + 1 .. phi, and the first ones that are kept
        cap = std::min<long>(cap, ((long)a.mask.window + h.z.per / a.rep + 1) / TLM_PAGE + 2 + mmi_cdiv(a.mask.keep, TLM_PAGE));
    cap = std::max(cap, 1l);
    const long units = std::max(1l, groups * a.c.kv_heads);
    const size_t each = (size_t)kv8_slots(a.q, h.z) * a.c.kv_heads * h.z.per * (a.c.vdim + 2);      // floats per split
    const size_t what = 4 * (size_t)kv8_slots(a.q, h.z);
    long most = room > what ? std::min<long>(KV8_MAX_SPLIT, (long)((room - what) / std::max<size_t>(1, each))) : 1;
    if (most < 2) most = 1;
    long per = std::max((cap * units + aim - 1) / aim, (cap + most - 1) / most);
    per = std::min((per + step - 1) / step * step, (cap + step - 1) / step * step);
    h.pages = (int)per;
    h.nsplit = (int)((cap + per - 1) / per);
    return h.nsplit > 1 ? each * h.nsplit + what : 0;
}

}  // namespace

int tlm_kv8_append(hipStream_t s, TlmKv8Append a, int dtype) {
    a.z = kv8_cut(a.q, 1, KV8_BLOCK, 2);               // (a portion of n rows touches at most (n + 14) / 16 + 1 blocks)
    const dim3 grid((unsigned)kv8_slots(a.q, a.z), mmi_cdiv(a.c.kv_heads, 4), 2);
    return by_codes(a.c.e4m3, [&](auto e) {
        const bool wide = a.c.dim > 128 || a.c.vdim > 128;
        if (dtype == MMI_F32 && wide) MMI_LAUNCH((k_tlm_kv8_append<float, decltype(e)::value, 256>), grid, 256, 0, s, a);
        else if (dtype == MMI_F32) MMI_LAUNCH((k_tlm_kv8_append<float, decltype(e)::value, 128>), grid, 256, 0, s, a);
        else if (wide) MMI_LAUNCH((k_tlm_kv8_append<uint16_t, decltype(e)::value, 256>), grid, 256, 0, s, a);
        else MMI_LAUNCH((k_tlm_kv8_append<uint16_t, decltype(e)::value, 128>), grid, 256, 0, s, a);
        MMI_CHECK_LAUNCH();
        return (int)MMI_OK;
    });
}

size_t tlm_kv8_plan(TlmKv8Attn& a, long cap, size_t room) {
    a.both = a.q.row0 != nullptr;
    a.few.z = Kv8Cut{0, 16, a.both ? 1 : mmi_cdiv(a.rep, 16), 0};
    a.few.cols = a.both ? KV8_FEW : std::min(16, a.rep);
    const size_t few = split_pages(a, a.few, kv8_slots(a.q, a.few.z), cap, room, KV8_WORKGROUPS, 4);      // (each of a workgroup's four waves takes every fourth page)
    if (!a.both) return few;
    a.many.z = Kv8Cut{a.rep, KV8_MANY, 1, 0};
    if ((long)a.q.T * a.rep / (KV8_FEW + 1) < a.q.n) a.many.z = Kv8Cut{a.rep, KV8_MANY, 0, KV8_FEW + 1};
    a.many.cols = KV8_MANY;
    const long full = (long)a.q.T * a.rep / KV8_MANY + 1;
    return few + split_pages(a, a.many, full + (kv8_slots(a.q, a.many.z) - full) / 4, cap, room - few, attn_bound(a.c) > 128 ? KV8_TILES_WIDE : KV8_TILES, 1);
}
void tlm_kv8_workspace(TlmKv8Attn& a, float* w) {
    for (Kv8Share* h : {&a.few, &a.many}) {
        if (h->nsplit <= 1) continue;
        const size_t parts = (size_t)kv8_slots(a.q, h->z) * a.c.kv_heads * h->nsplit * h->z.per;
        h->po = w;
        h->pml = w + parts * a.c.vdim;
        w += parts * (a.c.vdim + 2);
        h->what = (int*)w;
        w += 4 * kv8_slots(a.q, h->z);
    }
}

int tlm_kv8_attend(hipStream_t s, const TlmKv8Attn& a, int dtype, bool f32) {
    if (dtype == MMI_BF16) return launch_attn_d<uint16_t, TlmBf16, 1>(s, a);
    return f32 ? launch_attn_d<float, TlmF32, 2>(s, a) : launch_attn_d<float, TlmBf16, 1>(s, a);
}

extern "C" int mmi_kv_append(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                             int64_t v_head, mmi_stream stream) {
    TlmKv8Append a;
    memset(&a, 0, sizeof(a));
    int rc;
    if ((rc = check_cache(cache, &a.c, "mmi_kv_append")) || (rc = check_seqs(seqs, &a.q, "mmi_kv_append"))) return rc;
    if (!a.q.n || !a.q.T) return MMI_OK;
    if ((rc = check_rows(k, k_row, k_head, dtype, "mmi_kv_append")) || (rc = check_rows(v, v_row, v_head, dtype, "mmi_kv_append"))) return rc;
    a.k = k;
    a.v = v;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    a.wide = aligned4(k, k_row, k_head, dtype);
    return tlm_kv8_append((hipStream_t)stream, a, dtype);
}

extern "C" int mmi_kv_read(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, void* k, void* v, mmi_stream stream) {
    TlmKv8Read a;
    memset(&a, 0, sizeof(a));
    int rc;
    if ((rc = check_cache(cache, &a.c, "mmi_kv_read")) || (rc = check_seqs(seqs, &a.q, "mmi_kv_read"))) return rc;
    if (!a.q.n || !a.q.T) return MMI_OK;
    if ((rc = check_rows(k, 0, 0, dtype, "mmi_kv_read")) || (rc = check_rows(v, 0, 0, dtype, "mmi_kv_read"))) return rc;
    if (((uintptr_t)k | (uintptr_t)v) % 16) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_read: outputs must be aligned to 16 bytes");
    a.k = k;
    a.v = v;
    a.z = kv8_cut(a.q, 1, KV8_BLOCK, 2);
    return launch_read((hipStream_t)stream, a, dtype);
}

namespace {
int attn_args(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t heads, int32_t window, int32_t keep_first, TlmKv8Attn* a, size_t* floats) {
    memset(a, 0, sizeof(*a));
    int rc;
    if ((rc = check_cache(cache, &a->c, "mmi_kv_attend")) || (rc = check_seqs(seqs, &a->q, "mmi_kv_attend"))) return rc;
    if (heads < 1 || heads % cache->kv_heads || heads / cache->kv_heads > 1024) return mmi_fail(MMI_ERR_SHAPE, "mmi_kv_attend: query heads are a multiple of the key/value heads, at most 1024 times");
    if (window < 0 || keep_first < 0) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: negative window");
    a->rep = heads / cache->kv_heads;
    a->nd = cache->vdim / 16;
    a->mask = TlmMask{window, window > 0 ? std::min(keep_first, TLM_KEEP) : 0, 0.f};
    if ((long)a->q.T * a->rep > 1l << 26) return mmi_fail(MMI_ERR_SHAPE, "mmi_kv_attend: at most 2^26 rows times query heads of a group");
    *floats = tlm_kv8_plan(*a, seqs->n ? std::min(seqs->table_ld, 1 << 25) : 1, (size_t)1 << 30);      // (2^31 positions; twice a page's number has to stay in 31 bits)
    long groups = 0;
    for (const Kv8Share* h : {&a->few, &a->many})
        if (h->nsplit) groups += kv8_slots(a->q, h->z) * (long)cache->kv_heads * h->nsplit;
    if (groups > 1l << 23) return mmi_fail(MMI_ERR_SHAPE, "mmi_kv_attend: too many sequences, rows and heads for one call");      // (2^31 lanes a launch)
    return MMI_OK;
}
}  // namespace

extern "C" int64_t mmi_kv_attend_workspace(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t heads, int32_t window, int32_t keep_first) {
    TlmKv8Attn a;
    size_t floats;
    const int rc = attn_args(cache, seqs, heads, window, keep_first, &a, &floats);
    return rc ? rc : (int64_t)(floats * sizeof(float));
}

extern "C" int mmi_kv_attend(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, int32_t heads, const void* q, int64_t q_row, int64_t q_head, void* out,
                             int64_t out_row, int64_t out_head, float scale, int32_t window, int32_t keep_first, int32_t flags, void* workspace, int64_t workspace_bytes,
                             mmi_stream stream) {
    TlmKv8Attn a;
    size_t floats;
    int rc = attn_args(cache, seqs, heads, window, keep_first, &a, &floats);
    if (rc) return rc;
    if (!a.q.n || !a.q.T) return MMI_OK;
    if ((rc = check_rows(q, q_row, q_head, dtype, "mmi_kv_attend")) || (rc = check_rows(out, out_row, out_head, dtype, "mmi_kv_attend"))) return rc;
    if (!rows_apart(a.q.T, out_row, heads, out_head, a.c.vdim)) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: rows or heads of the output share memory");
    if (!aligned4(out, out_row, out_head, dtype)) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: four elements of the output must be aligned");
    if (flags & ~(MMI_KV_SINK | MMI_KV_ZERO_REST)) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: unknown flags");
    if (!(scale == scale) || scale - scale != 0.f) return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: the scale is not finite");
    if (floats && (!workspace || workspace_bytes < (int64_t)(floats * sizeof(float)) || (uintptr_t)workspace % 16))
        return mmi_fail(MMI_ERR_INVALID, "mmi_kv_attend: the workspace is too small (mmi_kv_attend_workspace) or not aligned to 16 bytes");
    a.x = q;
    a.x_row = q_row;
    a.x_head = q_head;
    a.wide = aligned4(q, q_row, q_head, dtype);
    a.out = out;
    a.out_row = out_row;
    a.out_head = out_head;
    a.mask.scale = scale * 1.44269504088896340736f;
    a.sink = flags & MMI_KV_SINK;
    a.rest = flags & MMI_KV_ZERO_REST;
    tlm_kv8_workspace(a, (float*)workspace);
    return tlm_kv8_attend((hipStream_t)stream, a, dtype, dtype == MMI_F32);
}

// ---- beam search ---------------------------------------------------------------------------------------------------------
namespace {
struct BeamSpace { size_t m, s, x, i, total; };            // where the parts of the workspace begin, in bytes
BeamSpace beam_space(int rows, int beams, int vocab) {
    const size_t lists = (size_t)rows * mmi_cdiv(vocab, BEAM_CHUNK);
    BeamSpace z;
    z.s = 0;
    z.m = lists * sizeof(double);
    z.x = z.m + lists * sizeof(float);
    z.i = z.x + lists * beams * sizeof(float);
    z.total = z.i + lists * beams * sizeof(int);
    return z;
}
int check_beams(int64_t batch, int32_t beams, int32_t vocab, const char* at) {
    if (batch < 0 || beams < 1 || vocab < 1) return mmi_fail(MMI_ERR_INVALID, std::string(at) + ": bad sizes");
    if (beams > BEAM_MAX) return mmi_fail(MMI_ERR_UNSUPPORTED, std::string(at) + ": at most 32 beams");
    if (batch * beams > 65535 || vocab > 1 << 20) return mmi_fail(MMI_ERR_SHAPE, std::string(at) + ": at most 65535 beams of all requests and 2^20 tokens");
    return MMI_OK;
}
}  // namespace

extern "C" int64_t mmi_beam_select_workspace(int32_t batch, int32_t beams, int32_t vocab) {
    const int rc = check_beams(batch, beams, vocab, "mmi_beam_select");
    return rc ? rc : (int64_t)beam_space(batch * beams, beams, vocab).total;
}

extern "C" int mmi_beam_select(int32_t batch, int32_t beams, int32_t vocab, int32_t dtype, const void* logits, int64_t row, const float* score, const int32_t* length,
                               const uint8_t* finished, int32_t eos, float length_penalty, float* out_score, int32_t* out_parent, int32_t* out_token, uint8_t* out_finished,
                               int32_t* out_length, void* workspace, int64_t workspace_bytes, mmi_stream stream) {
    int rc = check_beams(batch, beams, vocab, "mmi_beam_select");
    if (rc || !batch) return rc;
    if ((rc = check_rows(logits, row, 0, dtype, "mmi_beam_select"))) return rc;
    if (!score || !out_score || !out_parent || !out_token) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_select: null tensor");
    if (finished && (eos < 0 || eos >= vocab)) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_select: finished beams need an end token of the vocabulary");
    if (!(fabsf(length_penalty) <= BEAM_PENALTY)) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_select: a length penalty is between -16 and 16");
    if (length_penalty != 0.f && !length) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_select: a length penalty needs lengths");
    const BeamSpace z = beam_space(batch * beams, beams, vocab);
    if (!workspace || workspace_bytes < (int64_t)z.total || (uintptr_t)workspace % 16) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_select: the workspace is too small (mmi_beam_select_workspace) or not aligned to 16 bytes");
    char* w = (char*)workspace;
    TlmBeamArgs a;
    memset(&a, 0, sizeof(a));
    a.x = logits;
    a.ld = row;
    a.V = vocab;
    a.beams = beams;
    a.chunks = mmi_cdiv(vocab, BEAM_CHUNK);
    a.score = score;
    a.length = length;
    a.done = finished;
    a.eos = eos;
    a.alpha = (double)length_penalty;
    a.wm = (float*)(w + z.m);
    a.ws = (double*)(w + z.s);
    a.wx = (float*)(w + z.x);
    a.wi = (int*)(w + z.i);
    a.out_score = out_score;
    a.out_parent = out_parent;
    a.out_token = out_token;
    a.out_done = out_finished;
    a.out_length = out_length;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MMI_F32) MMI_LAUNCH((k_tlm_beam_rows<float>), dim3(mmi_cdiv(a.chunks, 4), batch * beams), 256, 0, s, a);
    else MMI_LAUNCH((k_tlm_beam_rows<uint16_t>), dim3(mmi_cdiv(a.chunks, 4), batch * beams), 256, 0, s, a);
    MMI_CHECK_LAUNCH();
    MMI_LAUNCH(k_tlm_beam_pick, batch, 256, 0, s, a);
    MMI_CHECK_LAUNCH();
    return MMI_OK;
}

namespace {
int reorder_unit(const TlmReorderTensor& t) {              // bytes that are moved at once
    const uintptr_t all = (uintptr_t)t.p | (uintptr_t)t.stride | (uintptr_t)t.bytes;
    return all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
}
}  // namespace

int tlm_reorder(hipStream_t s, int n, const TlmReorderTensor* tensors, int groups, int beams, const int* parent, const int* row) {
    for (int i = 0; i < n; ++i)                            // (before any of them has moved)
        if (tensors[i].bytes / reorder_unit(tensors[i]) > 0x3fffffffl) return mmi_fail(MMI_ERR_SHAPE, "reorder: a row is too long");
    for (int i = 0; i < n;) {
        TlmReorder a;
        memset(&a, 0, sizeof(a));
        a.beams = beams;
        a.parent = parent;
        a.row = row;
        unsigned blocks = 0;
        for (; i < n && a.n < BEAM_TENSORS; ++i) {
            const TlmReorderTensor& t = tensors[i];
            const int unit = reorder_unit(t);
            const long units = t.bytes / unit;
            if (!units) continue;
            const unsigned more = (unsigned)mmi_cdiv64(units, 256);
            if (blocks + more > 0x7fffffu) break;          // (2^31 lanes a launch)
            a.t[a.n++] = TlmReorder::T{(char*)t.p, (long)t.stride, (unsigned)units, blocks, unit};
            blocks += more;
        }
        if (!a.n) continue;
        const dim3 grid(blocks, (unsigned)groups);
        if (beams <= 4) MMI_LAUNCH((k_tlm_reorder<4>), grid, 256, 0, s, a);
        else if (beams <= 8) MMI_LAUNCH((k_tlm_reorder<8>), grid, 256, 0, s, a);
        else if (beams <= 16) MMI_LAUNCH((k_tlm_reorder<16>), grid, 256, 0, s, a);
        else MMI_LAUNCH((k_tlm_reorder<32>), grid, 256, 0, s, a);
        MMI_CHECK_LAUNCH();
    }
    return MMI_OK;
}

namespace {
// Does a byte of one tensor's rows belong to another's, or to the parents?  Tensors whose ranges overlap may be views of one buffer, a row of theirs
// being a part of its row: with strides that are equal they share nothing where the parts, modulo the stride, are apart.
bool rows_share_memory(std::vector<TlmReorderTensor> t, int rows, const TlmReorderTensor& parents) {
    auto end = [&](const TlmReorderTensor& x) { return (uintptr_t)x.p + (uintptr_t)x.stride * (uintptr_t)(rows - 1) + (uintptr_t)x.bytes; };
    t.erase(std::remove_if(t.begin(), t.end(), [](const TlmReorderTensor& x) { return x.bytes == 0; }), t.end());
    for (const TlmReorderTensor& x : t) {                  // (the parents' first byte behind x's start: in or behind its row k)
        const uintptr_t a = (uintptr_t)parents.p, b = a + (uintptr_t)parents.bytes, p = (uintptr_t)x.p;
        if (b <= p || a >= end(x)) continue;
        const uintptr_t k = a < p ? 0 : std::min<uintptr_t>((a - p) / (uintptr_t)x.stride, (uintptr_t)rows - 1), row = p + k * (uintptr_t)x.stride;
        if (a < row + (uintptr_t)x.bytes || (k + 1 < (uintptr_t)rows && b > row + (uintptr_t)x.stride)) return true;
    }
    std::sort(t.begin(), t.end(), [](const TlmReorderTensor& x, const TlmReorderTensor& y) { return (uintptr_t)x.p < (uintptr_t)y.p; });
    for (size_t i = 0; i < t.size();) {                    // a cluster: ranges that overlap one another in a chain
        size_t j = i + 1;
        for (uintptr_t to = end(t[i]); j < t.size() && (uintptr_t)t[j].p < to; ++j) to = std::max(to, end(t[j]));
        if (j > i + 1) {
            const uintptr_t stride = (uintptr_t)t[i].stride, from = (uintptr_t)t[i].p;
            std::vector<std::pair<uintptr_t, uintptr_t>> part;
            for (size_t k = i; k < j; ++k) {
                if ((uintptr_t)t[k].stride != stride) return true;
                const uintptr_t at = ((uintptr_t)t[k].p - from) % stride;
                part.push_back({at, at + (uintptr_t)t[k].bytes});
            }
            std::sort(part.begin(), part.end());
            for (size_t k = 1; k < part.size(); ++k)
                if (part[k].first < part[k - 1].second) return true;
            if (part.back().second > stride + part[0].first) return true;
        }
        i = j;
    }
    return false;
}
}  // namespace

extern "C" int mmi_beam_reorder(int32_t n, void* const* tensors, const int64_t* strides, const int64_t* row_bytes, int32_t batch, int32_t beams, const int32_t* parents,
                                mmi_stream stream) {
    int rc = check_beams(batch, beams, 1, "mmi_beam_reorder");
    if (rc || !batch || !n) return rc;
    if (n < 0 || !tensors || !strides || !row_bytes || !parents) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_reorder: null argument");
    if (n > 1 << 16) return mmi_fail(MMI_ERR_SHAPE, "mmi_beam_reorder: at most 2^16 tensors");
    const int rows = batch * beams;
    std::vector<TlmReorderTensor> t((size_t)n);
    for (int i = 0; i < n; ++i) {
        if (!tensors[i] || row_bytes[i] < 0 || strides[i] < row_bytes[i]) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_reorder: rows are apart and not null");
        if (strides[i] > (int64_t)1 << 46) return mmi_fail(MMI_ERR_SHAPE, "mmi_beam_reorder: rows are too far apart");      // (65535 of them within 2^62)
        t[i] = TlmReorderTensor{tensors[i], strides[i], row_bytes[i]};
    }
    // (a tensor given twice would be read and written by two workgroups, parents among the rows read by some behind others' writes)
    if (rows_share_memory(t, rows, TlmReorderTensor{(void*)parents, 4ll * rows, 4ll * rows})) return mmi_fail(MMI_ERR_INVALID, "mmi_beam_reorder: two tensors share memory");
    return tlm_reorder((hipStream_t)stream, n, t.data(), batch, beams, parents, nullptr);
}
