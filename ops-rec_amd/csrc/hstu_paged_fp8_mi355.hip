// C ABI of the 8-bit paged cache (include/hstu_mi355.h): argument checks, choice of the kernel variant, launch.
#include "../../include/hstu_mi355.h"

#include <hip/hip_runtime.h>

#include <algorithm>

#include "hstu_error.h"
#include "hstu_paged_fp8_append_kernel.hip.h"
#include "hstu_paged_fp8_evict_kernel.hip.h"
#include "hstu_paged_fp8_join_kernel.hip.h"
#include "hstu_paged_fp8_variants.h"

namespace {

using namespace hstu;

constexpr int kBlock = kFp8Block;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_cache(const hstu_paged_fp8_cache& c)
{
    if (c.k_cache == nullptr || c.v_cache == nullptr || c.k_scale == nullptr || c.v_scale == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "k_cache, v_cache, k_scale and v_scale must all be given");
    }
    if (c.cache_len == nullptr || c.page_offsets == nullptr || (c.page_ids == nullptr && c.n_page_ids > 0)) {
        return set_error(HSTU_ERR_NULLPTR, "cache_len, page_offsets and page_ids must all be given");
    }
    if (c.n_offsets < 2 || c.n_offsets - 1 > HSTU_MAX_BATCH) {
        return set_error(HSTU_ERR_INVALID, "batchSize limit (0, %d], but get %lld", HSTU_MAX_BATCH, (long long)(c.n_offsets - 1));
    }
    if (c.index_dtype != HSTU_IDX_I32 && c.index_dtype != HSTU_IDX_I64) {
        return set_error(HSTU_ERR_INVALID, "index dtype %d is not int32 or int64", c.index_dtype);
    }
    if (c.num_heads_k < 1 || c.num_heads_k > HSTU_MAX_HEADS) {
        return set_error(HSTU_ERR_INVALID, "head num expect in [1, %d], but the cache has %lld", HSTU_MAX_HEADS, (long long)c.num_heads_k);
    }
    if (c.head_dim < 16 || c.head_dim > HSTU_PAGED_FP8_MAX_HEAD_DIM || c.head_dim % 16 != 0) {
        return set_error(HSTU_ERR_INVALID, "headDim of the 8-bit cache expect a multiple of 16 in [16, %d], but value is %lld",
                         HSTU_PAGED_FP8_MAX_HEAD_DIM, (long long)c.head_dim);
    }
    if (c.page_size < kBlock || c.page_size % kBlock != 0 || c.page_size > HSTU_PAGED_FP8_MAX_SEQ_LEN_K) {
        return set_error(HSTU_ERR_INVALID, "page_size expect a multiple of %d, but value is %lld", kBlock, (long long)c.page_size);
    }
    if (c.num_pages < 1 || c.num_pages > INT32_MAX || c.n_page_ids < 0 || c.n_page_ids > INT32_MAX) {
        return set_error(HSTU_ERR_INVALID, "num_pages expect in [1, 2^31), n_page_ids in [0, 2^31), but they are %lld and %lld",
                         (long long)c.num_pages, (long long)c.n_page_ids);
    }
    if (c.num_pages * c.num_heads_k * (c.page_size / kBlock) > INT32_MAX) {
        return set_error(HSTU_ERR_INVALID, "the cache has more than 2^31 - 1 blocks of %d tokens and head", kBlock);
    }
    if (!aligned16(c.k_cache) || !aligned16(c.v_cache) || !aligned16(c.weights)) {
        return set_error(HSTU_ERR_INVALID, "k_cache, v_cache and weights must be 16-byte aligned");
    }
    return HSTU_OK;
}

Fp8Cache describe(const hstu_paged_fp8_cache& c)
{
    Fp8Cache r;
    r.k = static_cast<uint8_t*>(c.k_cache);
    r.v = static_cast<uint8_t*>(c.v_cache);
    r.k_scale = c.k_scale;
    r.v_scale = c.v_scale;
    r.weights = c.weights;
    r.cache_len = c.cache_len;
    r.page_offsets = c.page_offsets;
    r.page_ids = c.page_ids;
    r.n_batch = static_cast<int>(c.n_offsets - 1);
    r.n_heads = static_cast<int>(c.num_heads_k);
    r.dim = static_cast<int>(c.head_dim);
    r.blocks_per_page = static_cast<int>(c.page_size / kBlock);
    r.num_pages = static_cast<int>(c.num_pages);
    r.n_page_ids = static_cast<int>(c.n_page_ids);
    r.idx64 = c.index_dtype == HSTU_IDX_I64 ? 1 : 0;
    return r;
}

int launched(const char* name)
{
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HSTU_OK : set_error(HSTU_ERR_RUNTIME, "launch of %s failed: %s", name, hipGetErrorString(err));
}

bool is_16bit(int dtype) { return dtype == HSTU_DT_BF16 || dtype == HSTU_DT_FP16; }

bool bad_max_keys(int64_t n) { return n < 1 || n > HSTU_PAGED_FP8_MAX_SEQ_LEN_K; }

// -------------------------------------------------------------------------------------------------------- attention ----

int check_fwd(const hstu_paged_fp8_fwd_params* p)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(hstu_paged_fp8_fwd_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(hstu_paged_fp8_fwd_params));
    }
    const int rc = check_cache(p->cache);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (!is_16bit(p->dtype)) {
        return set_error(HSTU_ERR_INVALID, "dtype %d of q is not bf16 or fp16", p->dtype);
    }
    if (p->total_q < 0 || (p->total_q > 0 && (p->q == nullptr || p->out == nullptr)) || p->seq_offset == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "q, out and seq_offset must all be given");
    }
    if (!aligned16(p->q) || !aligned16(p->out)) {
        return set_error(HSTU_ERR_INVALID, "q and out must be 16-byte aligned");
    }
    if (p->num_heads_q < 1 || p->num_heads_q > HSTU_MAX_HEADS || p->num_heads_q % p->cache.num_heads_k != 0) {
        return set_error(HSTU_ERR_INVALID, "head num of q expect in [1, %d] and a multiple of the cache's, but they are %lld and %lld", HSTU_MAX_HEADS,
                         (long long)p->num_heads_q, (long long)p->cache.num_heads_k);
    }
    if (p->max_seq_len_q < 1 || p->max_seq_len_q > HSTU_MAX_SEQ_LEN) {
        return set_error(HSTU_ERR_INVALID, "maxSeqLen expect in [1, %d], but value is %lld", HSTU_MAX_SEQ_LEN, (long long)p->max_seq_len_q);
    }
    if (bad_max_keys(p->max_seq_len_k)) {
        return set_error(HSTU_ERR_INVALID, "maxSeqLenK expect in [1, %d], but value is %lld", HSTU_PAGED_FP8_MAX_SEQ_LEN_K, (long long)p->max_seq_len_k);
    }
    if (p->num_target != nullptr && (p->target_group_size < 1 || p->target_group_size > INT32_MAX / 2)) {
        return set_error(HSTU_ERR_INVALID, "targetGroupSize must be greater than 0 when numTarget is defined");
    }
    if (p->window < 0 || p->sinks < 0) {
        return set_error(HSTU_ERR_INVALID, "window and sinks must not be negative");
    }
    return HSTU_OK;
}

struct Plan {
    const Fp8AttendVariant* v;
    Fp8AttendArgs a;
    int64_t units, all_tiles;  // (part, key head) pairs, row tiles
    uint64_t partial_bytes, join_bytes, weight_bytes;
    bool split;  // some sequence may have more than one part
    uint64_t bytes() const { return partial_bytes + join_bytes + weight_bytes; }
};

// Which variant, and how the keys of a tile are dealt to workgroups.
Plan plan(const hstu_paged_fp8_fwd_params* p)
{
    Plan r;
    const int64_t ratio = p->num_heads_q / p->cache.num_heads_k, rows = p->max_seq_len_q * ratio;
    const int64_t pairs = (p->cache.n_offsets - 1) * p->cache.num_heads_k;
    int groups = 0;
    while (kFp8Groups[groups] * 32 < p->cache.head_dim) {
        ++groups;
    }
    const Fp8AttendTable& table = p->dtype == HSTU_DT_BF16 ? kFp8AttendBf16 : kFp8AttendF16;
    // A workgroup's wavefronts share the keys of a tile of 32 rows, each converting what it reads: as many of them as a CU's registers take,
    // or half as many where there are more tiles than places for whole ones, so that one starts while another works (64 x 4 pairs of
    // 33 .. 40 rows on 200 .. 400 keys 14 us and 20 in whole ones, on 1500 .. 3000 38 and 45; of 8 .. 16 on 1500 .. 3000, as many tiles as
    // places, 31 and 32; 32 x 4 of them on 500 .. 1500 21 and 17).  Where tiles of 128 rows fill the machine their wavefronts share the
    // conversion (16 x 4 of 1024 rows on 2048 .. 8192 keys 237 us, 272 in tiles of 32; 24 x 4 of 512 on 2000 .. 8000 207 and 207, 64 x 4
    // on 1000 .. 3000 232 and 258; fp16 252 and 287, 219 and 219, 255 and 270): at 97 .. 128 dims and
    // without weights only, elsewhere it is the other way round (d 96 191 and 189, d 64 165 and 139, with weights 329 and 307).
    const bool narrow = groups < 2;  // up to 64 dims a CU's registers take two workgroups
    const bool weights = p->cache.weights != nullptr, by_tile = groups == 3 && !weights && pairs * (rows / kFp8TileRows) >= 512;
    const bool half = pairs * ceil_div(rows, kFp8KeysRows) > (narrow ? 512 : 256);
    r.v = by_tile ? &table.tile : &table.keys[groups][half ? 1 : 0][weights ? 1 : 0];
    Fp8AttendArgs& a = r.a;
    a.c = describe(p->cache);
    a.q = p->q;
    a.offs_q = p->seq_offset;
    a.num_target = p->num_target;
    a.out = p->out;
    a.partial = nullptr;
    a.joins = nullptr;
    a.weight_partial = nullptr;
    a.total_q = p->total_q;
    a.n_heads_q = static_cast<int>(p->num_heads_q);
    a.ratio = static_cast<int>(ratio);
    a.max_q = static_cast<int>(p->max_seq_len_q);
    a.max_k = static_cast<int>(p->max_seq_len_k);
    a.group = static_cast<int>(p->num_target != nullptr ? p->target_group_size : 0);
    a.window = static_cast<int>(std::min<int64_t>(p->window, HSTU_PAGED_FP8_MAX_SEQ_LEN_K));
    a.sinks = static_cast<int>(p->window > 0 ? std::min<int64_t>(p->sinks, HSTU_PAGED_FP8_MAX_SEQ_LEN_K) : 0);
    a.c_exp = static_cast<float>(-p->alpha * 1.4426950408889634);
    a.c_out = static_cast<float>(p->alpha * p->silu_scale);
    a.row_tiles = static_cast<int>(ceil_div(rows, r.v->tile_rows));
    a.tile_first = 0;
    a.max_blocks = static_cast<int>(ceil_div(p->max_seq_len_k, kBlock));
    a.most_blocks = a.max_blocks;
    if (a.window > 0) {
        const int64_t seen = ceil_div(a.window + r.v->tile_rows / ratio, kBlock) + 2 + ceil_div(a.sinks, kBlock);
        a.most_blocks = static_cast<int>(std::min<int64_t>(a.most_blocks, seen));
    }
    // Parts (fp8_deal), where there are fewer workgroups than the machine has places, by the registers of the variants.  More cost more
    // than they spare: 24 x 4 pairs of up to 8 rows on 2000 .. 8000 keys 45 us without, 32 in 256, 39 in 512; 2 x 4 pairs, d 256, of up to
    // 256 rows 71, 37 and 46.  Nor are parts of a few blocks worth their sums: 2 x 4 pairs, d 64, on 500 .. 1500 keys 10 us without and 14 in
    // parts, on 2000 .. 8000 26 and 18.
    const int64_t batch = p->cache.n_offsets - 1, per_part = p->cache.num_heads_k * a.row_tiles;
    const int64_t total = (by_tile ? 1024 : 256) / per_part;
    const int least = by_tile ? 32 : 4 * (r.v->threads / 64);
    a.total_parts = 0;
    a.parts = 1;
    a.chunk = a.most_blocks;
    if (2 * total >= 3 * batch && a.most_blocks > 2 * least) {
        if (batch <= 64) {
            a.chunk = least;
            a.total_parts = static_cast<int>(total);
        } else {
            a.parts = static_cast<int>(std::min(ceil_div(total, batch), ceil_div(a.most_blocks, least)));
            a.chunk = static_cast<int>(ceil_div(a.most_blocks, a.parts));
            a.total_parts = static_cast<int>(batch * a.parts);
        }
    } else if ((by_tile || (half && a.most_blocks >= 128)) && batch <= 64) {
        // one part each, the longest sequences first: where workgroups follow one another and a late long one is waited for (24 x 4 pairs of
        // 50 .. 250 rows on 2000 .. 8000 keys, d 128, 86 us and 92 in the order they come in; on 500 .. 1500, where looking costs more, 32 and 29)
        a.total_parts = static_cast<int>(batch + 1);
    }
    r.split = a.chunk < a.most_blocks;
    r.partial_bytes = r.split ? static_cast<uint64_t>(a.total_parts) * per_part * r.v->tile_rows * p->cache.head_dim * 4 : 0;
    // A launch takes as many row tiles as its sums of weights have room for in 512 MiB, and as a grid holds; the others follow in launches
    // of their own.
    const uint64_t tile_bytes = static_cast<uint64_t>(pairs) * a.max_blocks * kBlock * 4;
    const int64_t units = (a.total_parts > 0 ? a.total_parts : batch) * p->cache.num_heads_k;
    r.all_tiles = a.row_tiles;
    a.row_tiles = static_cast<int>(std::min<int64_t>(a.row_tiles, std::max<int64_t>(kFp8MostSlots / (units + 7), 1)));
    if (weights) {
        a.row_tiles = static_cast<int>(std::min<int64_t>(a.row_tiles, std::max<int64_t>(static_cast<int64_t>(kFp8WeightBytes / tile_bytes), 1)));
    }
    r.units = units;
    r.join_bytes = r.split ? static_cast<uint64_t>(ceil_div(pairs * a.row_tiles, 2)) * 16 : 0;
    r.weight_bytes = weights && a.row_tiles > 1 ? a.row_tiles * tile_bytes : 0;
    return r;
}

// ---------------------------------------------------------------------------------------------------------- append ----

using AppendKernel = void (*)(const Fp8AppendArgs);
// by type and head dims up to 64, 128, 256: what a lane holds
const AppendKernel kAppend[2][3] = {
    {hstu_paged_fp8_append_kernel<bf16_tag, 64>, hstu_paged_fp8_append_kernel<bf16_tag, 128>, hstu_paged_fp8_append_kernel<bf16_tag, 256>},
    {hstu_paged_fp8_append_kernel<f16_tag, 64>, hstu_paged_fp8_append_kernel<f16_tag, 128>, hstu_paged_fp8_append_kernel<f16_tag, 256>},
};
int dim_slot(int64_t dim) { return dim <= 64 ? 0 : (dim <= 128 ? 1 : 2); }

bool bad_stride(int64_t s) { return s < 0 || s % 8 != 0; }

// ---------------------------------------------------------------------------------------------------------- evict ----

using EvictKernel = void (*)(const Fp8EvictArgs);
const EvictKernel kSelect = hstu_paged_fp8_select_kernel<1024, kFp8SelectKeys>, kSelectFew = hstu_paged_fp8_select_kernel<256, kFp8SelectFew + 8>;
const EvictKernel kMove[3] = {hstu_paged_fp8_move_kernel<64>, hstu_paged_fp8_move_kernel<128>, hstu_paged_fp8_move_kernel<256>};

int check_evict(const hstu_paged_fp8_evict_params* p)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(hstu_paged_fp8_evict_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(hstu_paged_fp8_evict_params));
    }
    const int rc = check_cache(p->cache);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->cache.weights == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "eviction goes by weights, which must be given");
    }
    if (p->new_page_offsets == nullptr || (p->new_page_ids == nullptr && p->n_new_page_ids > 0) || p->new_cache_len == nullptr || p->kept == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "new_page_offsets, new_page_ids, new_cache_len and kept must all be given");
    }
    if (p->n_new_page_ids < 0 || p->n_new_page_ids > INT32_MAX) {
        return set_error(HSTU_ERR_INVALID, "n_new_page_ids expect in [0, 2^31), but value is %lld", (long long)p->n_new_page_ids);
    }
    if (bad_max_keys(p->max_seq_len_k)) {
        return set_error(HSTU_ERR_INVALID, "maxSeqLenK expect in [1, %d], but value is %lld", HSTU_PAGED_FP8_MAX_SEQ_LEN_K, (long long)p->max_seq_len_k);
    }
    if (bad_max_keys(p->keep)) {
        return set_error(HSTU_ERR_INVALID, "keep expect in [1, %d], but value is %lld", HSTU_PAGED_FP8_MAX_SEQ_LEN_K, (long long)p->keep);
    }
    if (p->sinks < 0 || p->recent < 0) {
        return set_error(HSTU_ERR_INVALID, "sinks and recent must not be negative");
    }
    return HSTU_OK;
}

// rows that a sequence has at most: as many as are allowed, or as all the pages hold
int64_t evict_rows(const hstu_paged_fp8_evict_params* p) { return std::min(p->max_seq_len_k, p->cache.n_page_ids * p->cache.page_size); }
// scores of the longest sequence, in whole fours and where its first may be rounded down; none where LDS holds them
int64_t evict_pitch(const hstu_paged_fp8_evict_params* p) { return evict_rows(p) + 8 <= kFp8SelectKeys ? 0 : ceil_div(evict_rows(p), 4) * 4 + 8; }
uint64_t evict_workspace(const hstu_paged_fp8_evict_params* p) { return static_cast<uint64_t>(p->cache.n_offsets - 1) * evict_pitch(p) * 4; }

}  // namespace

extern "C" {

HSTU_API int hstu_paged_fp8_fwd_workspace_size(const hstu_paged_fp8_fwd_params* p, uint64_t* bytes)
{
    const int rc = check_fwd(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "workspace_bytes is NULL");
    }
    const Plan r = plan(p);
    *bytes = r.bytes();
    return HSTU_OK;
}

HSTU_API const char* hstu_paged_fp8_fwd_kernel_name(const hstu_paged_fp8_fwd_params* p) { return check_fwd(p) == HSTU_OK ? plan(p).v->name : nullptr; }

HSTU_API int hstu_paged_fp8_fwd(const hstu_paged_fp8_fwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream)
{
    const int rc = check_fwd(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->total_q == 0) {
        return HSTU_OK;
    }
    Plan r = plan(p);
    Fp8AttendArgs& a = r.a;
    if (r.bytes() > 0) {
        if (workspace == nullptr || workspace_bytes < r.bytes()) {
            return set_error(HSTU_ERR_WORKSPACE, "workspace of %llu bytes, %llu are needed", (unsigned long long)(workspace ? workspace_bytes : 0),
                             (unsigned long long)r.bytes());
        }
        if (!aligned16(workspace)) {
            return set_error(HSTU_ERR_INVALID, "workspace must be 16-byte aligned");
        }
        a.partial = r.partial_bytes > 0 ? static_cast<float*>(workspace) : nullptr;
        uint8_t* const joins = static_cast<uint8_t*>(workspace) + r.partial_bytes;
        a.joins = r.join_bytes > 0 ? reinterpret_cast<int2*>(joins) : nullptr;
        a.weight_partial = r.weight_bytes > 0 ? reinterpret_cast<float*>(joins + r.join_bytes) : nullptr;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned pairs = static_cast<unsigned>(a.c.n_batch) * a.c.n_heads;
    for (const int tiles = a.row_tiles; a.tile_first < r.all_tiles; a.tile_first += tiles) {
        a.row_tiles = static_cast<int>(std::min<int64_t>(tiles, r.all_tiles - a.tile_first));
        const int64_t slots = a.row_tiles == 1 ? r.units : ceil_div(r.units, 8) * 8 * a.row_tiles;
        hipLaunchKernelGGL(r.v->kernel, dim3(static_cast<unsigned>(slots)), dim3(r.v->threads), 0, s, a);
        if (r.split) {
            const auto join = p->dtype == HSTU_DT_BF16 ? hstu_paged_fp8_join_kernel<bf16_tag> : hstu_paged_fp8_join_kernel<f16_tag>;
            const int64_t most = ceil_div(static_cast<int64_t>(r.v->tile_rows) * a.c.dim, 256),
                          enough = ceil_div(kFp8JoinEnough, static_cast<int64_t>(a.row_tiles) * pairs);
            hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(std::min(most, enough)), a.row_tiles, pairs), dim3(256), 0, s, a, r.v->tile_rows);
        }
        if (a.weight_partial != nullptr) {
            hipLaunchKernelGGL(hstu_paged_fp8_weights_kernel, dim3(static_cast<unsigned>(ceil_div(a.max_blocks, 8)), pairs), dim3(256), 0, s, a);
        }
    }
    return launched(r.v->name);
}

HSTU_API int hstu_paged_fp8_append(const hstu_paged_fp8_append_params* p, void* stream)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(hstu_paged_fp8_append_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(hstu_paged_fp8_append_params));
    }
    const int rc = check_cache(p->cache);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (!is_16bit(p->dtype)) {
        return set_error(HSTU_ERR_INVALID, "dtype %d of k and v is not bf16 or fp16", p->dtype);
    }
    if (p->total < 0 || (p->total > 0 && (p->k == nullptr || p->v == nullptr)) || p->seq_offset == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "k, v and seq_offset must all be given");
    }
    if (!aligned16(p->k) || !aligned16(p->v) || bad_stride(p->k_stride_row) || bad_stride(p->k_stride_head) || bad_stride(p->v_stride_row) ||
        bad_stride(p->v_stride_head)) {
        return set_error(HSTU_ERR_INVALID, "k and v must be 16-byte aligned, their strides multiples of 8 elements");
    }
    if (bad_max_keys(p->max_seq_len)) {
        return set_error(HSTU_ERR_INVALID, "maxSeqLen expect in [1, %d], but value is %lld", HSTU_PAGED_FP8_MAX_SEQ_LEN_K, (long long)p->max_seq_len);
    }
    if (p->total == 0) {
        return HSTU_OK;
    }
    Fp8AppendArgs a;
    a.c = describe(p->cache);
    a.k = p->k;
    a.v = p->v;
    a.offs = p->seq_offset;
    a.total = p->total;
    a.k_row = p->k_stride_row;
    a.k_head = p->k_stride_head;
    a.v_row = p->v_stride_row;
    a.v_head = p->v_stride_head;
    const int64_t most = std::min(p->max_seq_len, p->total);
    a.max_rows = static_cast<int>(most);
    // n rows that begin anywhere in a block touch at most so many.  The number of workgroups along a sequence is odd: they go to the eight
    // dies in turn, and by a multiple of eight the last ones of all the sequences, which the short ones do not need, would fall to the
    // same dies (32 of 16128 blocks in all: 158 us where 106 is usual)
    const int64_t blocks = ((most + 2 * kBlock - 2) / kBlock) | 1;
    hipLaunchKernelGGL(kAppend[p->dtype == HSTU_DT_BF16 ? 0 : 1][dim_slot(a.c.dim)],
                       dim3(static_cast<unsigned>(blocks), 2u * static_cast<unsigned>(a.c.n_heads), static_cast<unsigned>(a.c.n_batch)),
                       dim3(kFp8AppendThreads), 0, static_cast<hipStream_t>(stream), a);
    return launched("hstu_paged_fp8_append_kernel");
}

HSTU_API int hstu_paged_fp8_evict_workspace_size(const hstu_paged_fp8_evict_params* p, uint64_t* bytes)
{
    const int rc = check_evict(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "workspace_bytes is NULL");
    }
    *bytes = evict_workspace(p);
    return HSTU_OK;
}

HSTU_API int hstu_paged_fp8_evict(const hstu_paged_fp8_evict_params* p, void* workspace, uint64_t workspace_bytes, void* stream)
{
    const int rc = check_evict(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (evict_workspace(p) > 0 && (workspace == nullptr || workspace_bytes < evict_workspace(p))) {
        return set_error(HSTU_ERR_WORKSPACE, "workspace of %llu bytes, %llu are needed", (unsigned long long)(workspace ? workspace_bytes : 0),
                         (unsigned long long)evict_workspace(p));
    }
    Fp8EvictArgs a;
    a.c = describe(p->cache);
    a.new_page_offsets = p->new_page_offsets;
    a.new_page_ids = p->new_page_ids;
    a.new_len = p->new_cache_len;
    a.kept = p->kept;
    if (evict_workspace(p) > 0 && !aligned16(workspace)) {
        return set_error(HSTU_ERR_INVALID, "workspace must be 16-byte aligned");
    }
    a.keys = static_cast<uint32_t*>(workspace);
    a.key_pitch = evict_pitch(p);
    a.n_new_page_ids = static_cast<int>(p->n_new_page_ids);
    a.max_k = static_cast<int>(evict_rows(p));
    a.keep = static_cast<int>(p->keep);
    a.sinks = static_cast<int>(std::min<int64_t>(p->sinks, p->keep));
    a.recent = static_cast<int>(std::min<int64_t>(p->recent, p->keep));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool few = a.max_k <= kFp8SelectFew;
    const EvictKernel select = few ? kSelectFew : kSelect;
    hipLaunchKernelGGL(select, dim3(static_cast<unsigned>(a.c.n_batch)), dim3(few ? 256 : 1024), 0, s, a);
    const int64_t most = std::min({p->keep, evict_rows(p), p->n_new_page_ids * p->cache.page_size});
    if (most > 0) {
        hipLaunchKernelGGL(kMove[dim_slot(a.c.dim)],
                           dim3(static_cast<unsigned>(ceil_div(most, kBlock)), 2u * static_cast<unsigned>(a.c.n_heads), static_cast<unsigned>(a.c.n_batch)),
                           dim3(kFp8AppendThreads), 0, s, a);
    }
    return launched("hstu_paged_fp8_move_kernel");
}

}  // extern "C"
