// C ABI of the attention over a 4-bit paged cache (include/hstu_cache.h): checks, the cut into runs, launches.
#include "hstu_cache.h"

#include <algorithm>

#include "hstu_cache_host.h"
#include "hstu_paged_attention_kernel.h"

namespace {

struct Plan {
    int step;          // rows of the kernel for few (1, 2, 4 or 8), or 0
    int mt, rw;        // else: 16-row tiles of a wave, waves that share out the rows
    int block, row_blocks, splits, run, share;
    int64_t workspace;
};

int check(const HstuPagedCache* c, const HstuPagedAttentionArgs* a, hstu::PagedAttentionParams& p) {
    const int rc = hstu_cache_fill(c, p.cache);
    if (rc) return rc;
    if (!a) return HSTU_ERR_NULL_POINTER;
    if (a->delta_size < 0 || a->max_seq_len <= 0 || a->q_heads <= 0 || a->q_heads % c->heads != 0) return HSTU_ERR_BAD_SHAPE;
    if (a->max_attn_len < 0 || a->contextual_seq_len < 0 || a->kv_splits < 0) return HSTU_ERR_BAD_SHAPE;
    if (c->dqk == 256 || c->dv == 256) {
        if (c->dqk != c->dv) return HSTU_ERR_BAD_HEAD_DIM;
    }
    if ((int64_t)a->delta_size * a->q_heads > (1 << 30) || (int64_t)c->batch * a->delta_size > (1ll << 31)) return HSTU_ERR_UNSUPPORTED;
    return 0;
}

Plan plan_of(const HstuPagedCache* c, const HstuPagedAttentionArgs* a) {
    Plan p{0, 1, 1, 16, 1, 1, 1, 4, 0};
    const int64_t rows = (int64_t)a->delta_size * (a->q_heads / c->heads);
    if (rows <= 8) {
        p.step = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
        p.block = p.step;
    } else {
        if (rows > 16) p.mt = c->dv == 256 ? 1 : 2;
        if (rows > 16 * p.mt) {
            p.rw = 4;
            // (blocks of 128 rows take 1.75 times as long as blocks of 64: 132 rows in three of 64 25 us, in two of 128 30)
            if (4 * ((rows + 63) / 64) < 7 * ((rows + 127) / 128)) p.mt = 1;
        }
        p.block = 16 * p.mt * p.rw;
    }
    p.row_blocks = (int)((rows + p.block - 1) / p.block);
    // (max_seq_len divides the result and may be far above what a row of the page table has room for)
    int64_t longest = std::min((int64_t)a->max_seq_len, (int64_t)c->table_columns * c->page_size);
    if (a->max_attn_len > 0 && (int64_t)a->max_attn_len + a->delta_size + a->contextual_seq_len < longest)
        longest = (int64_t)a->max_attn_len + a->delta_size + a->contextual_seq_len;
    const int64_t chunks = (longest + 31) / 32 + 1, wgs = (int64_t)p.row_blocks * c->heads * c->batch;
    // Runs of a step.  Joining costs 3 us, so sequences of up to 40 chunks are one run each (one of 512 positions: 8.0 us, in two runs 10.8; of 1024:
    // 10.3, in three 11.2), and so are those of up to 96 where they fill half of what the card holds, two workgroups of a CU (100 of up to 2048
    // positions and four heads: 22.3 us, in two runs 24.1).  Else runs that fill it once, for each begins with some microseconds of loads that wait
    // for each other (64 sequences of 1024 .. 4096 positions and four heads, 256 workgroups for whole sequences: in two runs 26.6 us, one 28.1, eight
    // 32.1); in eights, two chunks to each wave (33 sequences of up to 2048, four rows: runs of 16 17 us, of 18 18, whole sequences 20); none that
    // leaves a short second or third, which makes some of them up to 120 long; and else none longer than 96, so that the last of them do not run
    // alone (128 sequences of up to 16384 and eight heads: whole sequences 307 us, runs of 257 chunks 276, of 96 269, of 33 284).  Sequences of a few
    // chunks, more of them than fit, are a wave's each (1600 of up to 10 chunks, by workgroups, took a third longer).
    // More rows are split into equal parts of each sequence, of at least 8 or 16 chunks: what a part more costs is a partial sum of every row to
    // write and read.  Blocks: at least two workgroups of a CU, whose sequences are ranked.  Nine to 32 rows: parts that fill the card in one
    // round, 512 workgroups, or 256 of more than 16 rows of wide heads, whose waves need a SIMD each, or in two rounds where one would leave much of it empty (24 rows, 160 workgroups
    // for whole sequences of up to 8192: one part 88 us, two 74, three 64, four 67; 256 workgroups of up to 4096: one 49, two 57, four 66;
    // 16 rows, 128 workgroups of up to 8192: two 41, four 34, eight 37; 24 rows of 64 columns, the same: two 45, four 34, eight 35).
    const int64_t fill = (chunks * wgs + 511) / 512;
    int64_t run = 16;
    if (p.step) {
        if (a->kv_splits > 0) {
            run = (chunks + a->kv_splits - 1) / a->kv_splits;
        } else if (chunks <= 40 || (wgs >= 256 && chunks <= 96)) {
            run = chunks;
        } else {
            run = (fill + 4) / 8 * 8;
            if (run > 96) run = 96;
            if (run < 16) run = 16;
            if (chunks > run && chunks / run <= 2 && chunks % run <= run / 4) run = (chunks / (chunks / run) + 8) / 8 * 8;
        }
        if (run < 16) run = 16;
        if (run > chunks) run = chunks;
    } else {
        int64_t parts = a->kv_splits;
        if (parts == 0 && wgs > 0) {
            const int64_t slots = p.rw == 4 || p.mt == 1 || c->dqk + c->dv < 256 ? 512 : 256;
            parts = p.rw == 4 ? (slots + wgs - 1) / wgs : slots / wgs;
            if (p.rw != 4 && parts <= 2 && 2 * slots / wgs > 2 * parts) parts = 2 * slots / wgs;
        }
        if (p.rw == 4) run = 8;
        if (parts > (chunks + run - 1) / run) parts = (chunks + run - 1) / run;
        p.splits = parts < 1 ? 1 : (int)parts;
        if (run > chunks) run = chunks;
    }
    if (p.step && chunks <= 17 && wgs > 1024) p.share = 1, run = chunks;
    p.run = (int)run;
    if (p.step) p.splits = (int)((chunks + run - 1) / run);
    if (p.splits > 1) p.workspace = (int64_t)p.splits * c->batch * a->delta_size * a->q_heads * c->dv * 4;
    return p;
}

typedef std::integral_constant<int, 1> One;

template <class TT, int DK, int DV>
int launch_sized(const hstu::PagedAttentionParams& p, const Plan& plan, hipStream_t stream) {
    auto go = [&](auto mt) {
        hipLaunchKernelGGL((hstu::hstu_paged_attention_kernel<TT, DK, DV, decltype(mt)::value>), dim3((unsigned)p.items), dim3(256), 0, stream, p);
    };
    auto block = [&](auto mt) {
        hipLaunchKernelGGL((hstu::hstu_paged_block_kernel<TT, DK, DV, decltype(mt)::value>), dim3((unsigned)(p.items * (int64_t)plan.row_blocks)), dim3(256), 0, stream, p);
    };
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    auto step = [&](auto rp) {
        hipLaunchKernelGGL((hstu::hstu_paged_step_kernel<TT, DK, DV, decltype(rp)::value>), dim3((unsigned)((p.items * p.share + 3) / 4)), dim3(256), 0, stream, p);
    };
    if (plan.step == 1) step(One{});
    else if (plan.step == 2) step(Two{});
    else if (plan.step == 4) step(Four{});
    else if (plan.step == 8) step(std::integral_constant<int, 8>{});
    else if (plan.rw == 4 && plan.mt == 1) block(One{});
    else if (plan.mt == 1) go(One{});
    else if constexpr (DV != 256) {
        if (plan.rw == 4) block(Two{});
        else go(Two{});
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && p.splits > 1) {
        const int64_t total8 = p.partial_stride / 8;
        auto join = [&](auto parts) {
            constexpr int P = decltype(parts)::value;
            hipLaunchKernelGGL((hstu::hstu_paged_join_kernel<TT, P>), dim3((unsigned)((total8 * P + 255) / 256)), dim3(256), 0, stream, p, plan.block, total8);
        };
        if (p.splits > 4) join(std::integral_constant<int, 8>{});
        else join(One{});
        e = hipGetLastError();
    }
    if (e == hipSuccess) return 0;
    hstu_cache_set_last_error("paged attention kernel launch", (int)e);
    return HSTU_ERR_LAUNCH;
}

template <class TT>
int launch(const hstu::PagedAttentionParams& p, const Plan& plan, hipStream_t stream) {
    auto with_dv = [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        if (p.cache.dv == 32) return launch_sized<TT, DK, 32>(p, plan, stream);
        if (p.cache.dv == 64) return launch_sized<TT, DK, 64>(p, plan, stream);
        return launch_sized<TT, DK, 128>(p, plan, stream);
    };
    if (p.cache.dqk == 32) return with_dv(std::integral_constant<int, 32>{});
    if (p.cache.dqk == 64) return with_dv(std::integral_constant<int, 64>{});
    if (p.cache.dqk == 128) return with_dv(std::integral_constant<int, 128>{});
    return launch_sized<TT, 256, 256>(p, plan, stream);
}

}  // namespace

extern "C" {

size_t hstu_cache_attention_workspace_bytes(const HstuPagedCache* c, const HstuPagedAttentionArgs* a) {
    hstu::PagedAttentionParams p{};
    if (check(c, a, p) != 0 || c->batch == 0 || a->delta_size == 0) return 0;
    return (size_t)plan_of(c, a).workspace;
}

int hstu_cache_attention(const HstuPagedCache* c, const HstuPagedAttentionArgs* a, void* stream) {
    hstu::PagedAttentionParams p{};
    const int rc = check(c, a, p);
    if (rc) return rc;
    if (c->batch == 0 || a->delta_size == 0) return 0;
    if (c->pages == 0) return HSTU_ERR_BAD_SHAPE;
    if (c->pages > 2147483647) return HSTU_ERR_UNSUPPORTED;
    if (!a->q || !a->out || !a->seq_lengths || !c->page_table) return HSTU_ERR_NULL_POINTER;
    if (!hstu_cache_aligned(a->q) || !hstu_cache_aligned(a->out)) return HSTU_ERR_MISALIGNED;
    if (a->q_row_stride < 0 || a->q_head_stride < 0 || a->q_row_stride % 8 != 0 || a->q_head_stride % 8 != 0) return HSTU_ERR_MISALIGNED;
    const Plan plan = plan_of(c, a);
    if (plan.workspace > 0) {
        if (!a->workspace) return HSTU_ERR_NULL_POINTER;
        if (!hstu_cache_aligned(a->workspace)) return HSTU_ERR_MISALIGNED;
        if (a->workspace_bytes < plan.workspace) return HSTU_ERR_BAD_SHAPE;
    }
    const int64_t items = (int64_t)c->batch * c->heads * plan.splits;
    const int64_t joined = plan.splits > 1 ? (int64_t)c->batch * a->delta_size * a->q_heads * c->dv / 8 * (plan.splits > 4 ? 8 : 1) : 0;
    if (items * plan.row_blocks > kMaxBlocks || (joined + 255) / 256 > kMaxBlocks) return HSTU_ERR_UNSUPPORTED;
    if (!hstu_cache_device_is_gfx950()) return HSTU_ERR_BAD_DEVICE;
    p.q = (const char*)a->q, p.q_rs = a->q_row_stride, p.q_hs = a->q_head_stride, p.out = (char*)a->out;
    p.lengths = a->seq_lengths, p.lengths_i64 = a->seq_lengths_i64, p.targets = a->num_targets, p.targets_i64 = a->num_targets_i64;
    p.group = a->q_heads / c->heads, p.delta = a->delta_size, p.w = a->max_attn_len, p.c = a->contextual_seq_len;
    const float log2e = 1.4426950408889634f;
    p.c1 = -a->alpha * log2e, p.oscale = -1.f / (a->max_seq_len * log2e);
    p.row_blocks = plan.row_blocks, p.splits = plan.splits, p.run = plan.run, p.share = plan.share, p.items = (int)items;
    p.partial = (float*)a->workspace, p.partial_stride = (int64_t)c->batch * a->delta_size * a->q_heads * c->dv;
    return c->dtype == HSTU_BF16 ? launch<hstu::PagedBf16>(p, plan, (hipStream_t)stream) : launch<hstu::PagedF16>(p, plan, (hipStream_t)stream);
}

}  // extern "C"
