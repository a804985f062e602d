// attention_paged.hip — one query token a scene against a cache whose rows lie in pages.
//
// The kernel is gsv_cached.h's: a page holds a multiple of 16 rows, so 16 rows of a step have one page, whose
// first row is the base of their copy.  A table names the pages of a scene; a wave reads the entries of 32 of its
// steps by one load, 32 steps ahead.  Scenes of a batch differ in length, and their lengths are known on
// the device alone: every workgroup forms the pieces that the batch's rows are cut into, all of one
// size, and takes its own (paged_piece).
#include "gsv_cached.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

// One workgroup a scene and head; scenes of one part have their row already.
constexpr int kJoinWaves = 8;
template <typename T>
__global__ __launch_bounds__((64 * kJoinWaves)) void k_paged_join(const float *__restrict__ part_o,
                                                                  const float2 *__restrict__ part_ms,
                                                                  const int2 *__restrict__ parts, FastDiv by_heads,
                                                                  int heads, int dim, T *__restrict__ out) {
    const int row = blockIdx.x, s = fastdiv(row, by_heads), h = row - s * heads;
    const int2 p = parts[s];
    if (p.y == 1) return;
    join_row<T, kJoinWaves>(part_o, part_ms, (int64_t)p.x * heads + h, heads, p.y, dim, out + (int64_t)row * dim);
}

// Sets the workgroups of a key head that share a batch's steps: one round of them, as many as the CUs have room for
// at once.  Scenes of at most a step for each wave stay whole.
void paged_shares(const AttnArgs &a, int dtype, CacheArgs *c) {
    const int64_t size = dtype == GSV_BF16 ? 2 : 4, dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
    const int64_t waves = 512 / imax64(128, dp * size);
    c->splits = 1, c->shares = a.scenes;
    if (!a.scenes || a.k_tokens <= waves * kKeys) return;
    const int64_t lds = waves * (4 * kKeys * dp * size + (a.slopes ? 6 * kKeys * (size == 2 ? 16 : 4) : 0)) + 2048;
    const int64_t round = 256 * imin64(163840 / lds, 12 / waves);
    const int64_t most = ((int64_t)a.k_tokens + waves * kKeys - 1) / (waves * kKeys) * a.scenes;
    c->splits = 2;
    c->shares = (int)imax64(1, imin64(round / ((int64_t)a.kv_heads * c->head_tiles), most + a.scenes));
}

struct Paged {
    const AttnArgs &a;
    const CacheArgs &c;
    void *out;
    hipStream_t st;
    template <typename T, int DP, bool FAR, int CAP> void run() const {
        T *o = static_cast<T *>(out);
        const dim3 grid((unsigned)((int64_t)c.shares * a.kv_heads * c.head_tiles)), block(64 * kWaves<T, DP, kPieces>);
        if (a.scenes * 2 < c.shares) hipLaunchKernelGGL((k_attention_cached<T, DP, FAR, CAP, kPieces>), grid, block, 0, st, a, c, o);
        else hipLaunchKernelGGL((k_attention_cached<T, DP, FAR, CAP, kShares>), grid, block, 0, st, a, c, o);
        if (c.splits > 1)
            hipLaunchKernelGGL(k_paged_join<T>, dim3((unsigned)(a.scenes * a.heads)), dim3(64 * kJoinWaves), 0, st,
                               c.part_o, c.part_ms, c.parts, make_fastdiv(a.heads), a.heads, a.dim, o);
    }
};

int paged_plan(const gsv_attention *args, const gsv_pages *p, AttnArgs *a, CacheArgs *c) {
    if (!args || !p || args->causal || args->prefix || args->q_starts || args->k_starts ||
        args->scenes < 0 || args->scenes != args->q_tokens || p->pages < 1 || p->page_rows < kPageUnit ||
        p->page_rows % kPageUnit || p->table_pages < 0 || p->table_row < 0)
        return GSV_ERR_INVALID_ARGUMENT;
    const int64_t rows = (int64_t)p->page_rows * p->table_pages;
    if (rows > GSV_MAX_TOKENS) return GSV_ERR_SIZE_OVERFLOW;
    gsv_attention one = *args;
    one.scenes = 1;  // rows are addressed by scene and page here, not packed
    one.k = p->k, one.v = p->v, one.k_positions = p->positions, one.k_pos_row = p->pos_row;
    one.k_row = p->k_row, one.v_row = p->v_row, one.k_head = p->k_head, one.v_head = p->v_head;
    one.keep = p->keep, one.keep_bytes = p->keep_bytes;
    one.k_tokens = (int)rows;
    const int st = attention_args(&one, a);
    if (st != GSV_OK) return st;
    a->scenes = args->scenes;
    const int64_t tiles = (a->heads / a->kv_heads + kHeads - 1) / kHeads;
    if ((int64_t)a->scenes * a->kv_heads * tiles > (1 << 22) || (int64_t)a->scenes * a->heads >= (1 << 24))
        return GSV_ERR_SIZE_OVERFLOW;
    *c = CacheArgs{};
    c->head_tiles = (int)tiles;
    paged_shares(*a, args->dtype, c);
    return GSV_OK;
}

// The workspace: parts of the sums, their maxima and sums of weights, and which are a scene's.
struct Workspace {
    size_t rows, ms, parts, bytes;
};
Workspace paged_workspace(const AttnArgs &a, const CacheArgs &c) {
    if (c.splits == 1) return {};
    Workspace w;
    w.rows = ((size_t)c.shares + a.scenes) * a.heads;
    w.ms = w.rows * a.dim * sizeof(float);  // a multiple of 32 bytes
    w.parts = w.ms + w.rows * sizeof(float2);
    w.bytes = w.parts + a.scenes * sizeof(int2);
    return w;
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_attention_paged_workspace_bytes(const gsv_attention *args, const gsv_pages *pages,
                                                   size_t *bytes) {
    AttnArgs a;
    CacheArgs c;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = paged_plan(args, pages, &a, &c);
    if (st != GSV_OK) return st;
    *bytes = paged_workspace(a, c).bytes;
    return GSV_OK;
}

extern "C" int gsv_attention_paged(const gsv_attention *args, const gsv_pages *pages, const int32_t *lengths,
                                   void *out, void *workspace, size_t workspace_bytes, void *stream) {
    AttnArgs a;
    CacheArgs c;
    int st = paged_plan(args, pages, &a, &c);
    if (st != GSV_OK) return st;
    if (a.scenes == 0) return GSV_OK;
    const Workspace ws = paged_workspace(a, c);
    if (ws.bytes > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    const int64_t chunk = args->dtype == GSV_BF16 ? 8 : 4;
    c.k_scene = used_stride(pages->k_page, pages->pages);
    c.v_scene = used_stride(pages->v_page, pages->pages);
    if (!lengths || (pages->table_pages && !pages->table) || !out || (ws.bytes && !workspace) ||
        c.k_scene % chunk || c.v_scene % chunk || reinterpret_cast<uintptr_t>(out) % 16 ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
        return GSV_ERR_INVALID_ARGUMENT;
    c.lengths = lengths;
    c.k_pos_scene = pages->pos_page, c.keep_scene = pages->keep_page;
    c.part_o = static_cast<float *>(workspace);
    c.part_ms = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + ws.ms);
    c.parts = reinterpret_cast<int2 *>(static_cast<char *>(workspace) + ws.parts);
    c.table = pages->table, c.table_row = pages->table_row;
    c.pages = pages->pages, c.page_rows = pages->page_rows;
    c.by_rows = make_fastdiv(pages->page_rows);
    Paged f{a, c, out, as_stream(stream)};
    attention_variant(a, args->dtype, f);
    return check_launch();
}
