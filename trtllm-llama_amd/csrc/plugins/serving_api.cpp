// extern "C" surface of include/tllm_serving_api.h: every size, type, stride and alignment that a kernel relies on is checked here, on the host,
// before anything is launched.  What only the device knows (lengths, table entries, slots) the kernels check themselves.
#include "../kernels/serving_kernels.h"
#include <algorithm>
#include <exception>
#include <initializer_list>

using namespace tllm;
using namespace tllm::kernels;

namespace
{
bool is_page(int32_t v)
{
    return v == 16 || v == 32 || v == 64 || v == 128;
}

bool is_head(int32_t v)
{
    return v == 64 || v == 128 || v == 256;
}

bool aligned(const void* p, size_t to)
{
    return reinterpret_cast<uintptr_t>(p) % to == 0;
}

// `rows` pieces of `bytes`, one every `step` bytes
struct Range
{
    int64_t at, bytes, rows, step, end; // of the last piece
    Range(const void* p, int64_t bytes, int64_t rows = 1, int64_t step = 0)
        : at(static_cast<int64_t>(reinterpret_cast<uintptr_t>(p))), bytes(bytes), rows(bytes > 0 ? rows : 0), step(step)
    {
        if (rows > 1 && step < 0)
        {
            at += (rows - 1) * step;
            this->step = -step;
        }
        if (rows > 1 && this->step == bytes)
        {
            this->bytes *= rows;
            this->rows = 1;
        }
        if (this->rows <= 1)
            this->step = 0;
        end = at + (this->rows - 1) * this->step + this->bytes;
    }
    bool operator==(const Range& o) const { return at == o.at && bytes == o.bytes && rows == o.rows && step == o.step; }
};

int64_t floor_div(int64_t a, int64_t b)
{
    return a / b - (a % b < 0);
}

// a piece at `at` + k * step, first <= k <= last, reaches into [x, x + n)
bool meets(int64_t at, int64_t bytes, int64_t step, int64_t first, int64_t last, int64_t x, int64_t n)
{
    if (step == 0)
        return at < x + n && x < at + bytes;
    return std::max(first, floor_div(x - bytes - at, step) + 1) <= std::min(last, -floor_div(at - x - n, step) - 1);
}

bool pieces_meet(const Range& a, const Range& b)
{
    if (a.rows > b.rows)
        return pieces_meet(b, a);
    if (a.step == b.step) // only the distance counts
        return meets(b.at, b.bytes, b.step, 1 - a.rows, b.rows - 1, a.at, a.bytes);
    for (int64_t i = 0; i < a.rows; ++i)
        if (meets(b.at, b.bytes, b.step, 0, b.rows - 1, a.at + i * a.step, a.bytes))
            return true;
    return false;
}

inline bool overlap(const Range& a, const Range& b)
{
    return a.at < b.end && b.at < a.end && a.rows > 0 && b.rows > 0 && pieces_meet(a, b);
}

// [rows][heads][size] elements of 16 bits
struct Rows
{
    int64_t at, bytes, rows, step, heads, head_step;
    Rows(const void* p, int64_t rows, int64_t row, int32_t heads, int64_t head, int32_t size)
        : at(static_cast<int64_t>(reinterpret_cast<uintptr_t>(p))), bytes(2 * (int64_t) size), rows(rows), step(rows > 1 ? 2 * row : 0), heads(heads),
          head_step(heads > 1 ? 2 * head : 0)
    {
        if (heads > 1 && head_step == bytes)
        {
            bytes *= heads;
            this->heads = 1;
            head_step = 0;
        }
    }
    Range head(int64_t i) const { return Range(reinterpret_cast<const void*>(static_cast<uintptr_t>(at + i * head_step)), bytes, rows, step); }
    Range all() const
    {
        const int64_t r = (rows - 1) * step, h = (heads - 1) * head_step, low = at + std::min<int64_t>(r, 0) + std::min<int64_t>(h, 0);
        return Range(reinterpret_cast<const void*>(static_cast<uintptr_t>(low)), std::max(r, -r) + std::max(h, -h) + bytes);
    }
    bool operator==(const Rows& o) const { return at == o.at && bytes == o.bytes && rows == o.rows && step == o.step && heads == o.heads && head_step == o.head_step; }
};

bool overlap(const Rows& a, const Rows& b)
{
    if (!overlap(a.all(), b.all()))
        return false;
    const bool apart = a.head_step == b.head_step; // only the distance counts
    for (int64_t i = 0; i < (apart ? 1 : a.heads); ++i)
        for (int64_t j = apart ? 1 - a.heads : 0; j < b.heads; ++j)
            if (overlap(a.head(i), b.head(j)))
                return true;
    return false;
}

bool folded(const Rows& a) // two of its rows or heads share a place
{
    const Range first = a.head(0);
    if (first.rows > 1 && first.step < first.bytes)
        return true;
    for (int64_t i = 1; i < a.heads; ++i)
        if (overlap(first, a.head(i)))
            return true;
    return false;
}

constexpr int32_t kMaxRows = 1 << 19, kMaxHeads = 1024, kMaxTiles = 1 << 25;

#define TLLM_REFUSE(cond, ...)                                                                                         \
    do                                                                                                                 \
    {                                                                                                                  \
        if (cond)                                                                                                      \
        {                                                                                                              \
            set_error(__VA_ARGS__);                                                                                    \
            return false;                                                                                              \
        }                                                                                                              \
    } while (0)

bool plan_fits(const tllm_paged_plan_params_t* p)
{
    const char* const me = "tllm_paged_plan";
    TLLM_REFUSE(!p, "%s: null parameters", me);
    TLLM_REFUSE(p->n_seqs < 1 || p->n_seqs > kPlanMaxSeqs, "%s: n_seqs %d outside [1, %d]", me, p->n_seqs, kPlanMaxSeqs);
    TLLM_REFUSE(p->n_rows < 0 || p->n_rows > kMaxRows, "%s: n_rows %d outside [0, %d]", me, p->n_rows, kMaxRows);
    TLLM_REFUSE(!is_page(p->page_size), "%s: page_size %d is none of 16, 32, 64, 128", me, p->page_size);
    TLLM_REFUSE(p->num_blocks < 1 || (int64_t) p->num_blocks * p->page_size > INT32_MAX, "%s: num_blocks %d: 1 or more, times page_size below 2^31", me, p->num_blocks);
    TLLM_REFUSE(p->max_blocks < 1 || p->max_blocks > kMaxRows, "%s: max_blocks %d outside [1, %d]", me, p->max_blocks, kMaxRows);
    TLLM_REFUSE(p->table_stride < p->max_blocks, "%s: table_stride %lld is less than max_blocks %d", me, (long long) p->table_stride, p->max_blocks);
    TLLM_REFUSE(!p->lens || !p->new_lens || !p->ring || !p->ring_state || !p->block_table || !p->cu_tokens || !p->lens_out || !p->ring_state_out || !p->status
            || (p->n_rows && (!p->slot_map || !p->positions)),
        "%s: null tensor", me);
    for (const void* t : std::initializer_list<const void*>{p->lens, p->new_lens, p->ring, p->ring_state, p->block_table, p->cu_tokens, p->slot_map, p->positions, p->lens_out,
             p->ring_state_out, p->status})
        TLLM_REFUSE(!aligned(t, 4), "%s: a tensor is not 4-byte aligned", me);
    // several workgroups read what one of them writes, unless it is the whole of the same state
    const int64_t n = p->n_seqs * 4, rows = p->n_rows * 4;
    const Range lens(p->lens, n), state(p->ring_state, 8), lens_out(p->lens_out, n), state_out(p->ring_state_out, 8);
    const Range reads[] = {lens, {p->new_lens, n}, state};
    const Range writes[] = {lens_out, state_out, {p->cu_tokens, n + 4}, {p->slot_map, rows}, {p->positions, rows}, {p->status, 4}, {p->ring, (int64_t) p->num_blocks * 4},
        {p->block_table, (int64_t) p->max_blocks * 4, p->n_seqs, p->table_stride * 4}};
    for (const Range& w : writes)
    {
        for (const Range& r : reads)
            TLLM_REFUSE(overlap(w, r) && !((&w == &writes[0] && &r == &reads[0] && w == r) || (&w == &writes[1] && &r == &reads[2] && w == r)),
                "%s: a result lies where another tensor does", me);
        for (const Range& o : writes)
            TLLM_REFUSE(&o < &w && overlap(w, o), "%s: a result lies where another tensor does", me);
    }
    return true;
}

bool rows_fit(const char* me, const char* what, const void* t, int64_t row, int64_t head)
{
    TLLM_REFUSE(!t, "%s: null %s", me, what);
    TLLM_REFUSE(!aligned(t, 16) || row % 8 || head % 8, "%s: %s has to be 16-byte aligned, with strides that are multiples of 8 elements", me, what);
    return true;
}

bool cache_fits(const char* me, int32_t dtype, int32_t cache_type, int32_t head_size, int32_t page_size, int32_t num_blocks, int32_t kv_heads, const void* pool, const float* scales)
{
    TLLM_REFUSE(dtype != TLLM_HALF && dtype != TLLM_BF16, "%s: dtype %d is neither float16 nor bfloat16", me, dtype);
    TLLM_REFUSE(cache_type != TLLM_INT8 && cache_type != TLLM_FP8, "%s: cache_type %d is neither int8 nor fp8", me, cache_type);
    TLLM_REFUSE(!is_head(head_size), "%s: head_size %d is none of 64, 128, 256", me, head_size);
    TLLM_REFUSE(!is_page(page_size), "%s: page_size %d is none of 16, 32, 64, 128", me, page_size);
    TLLM_REFUSE(num_blocks < 1 || (int64_t) num_blocks * page_size > INT32_MAX, "%s: num_blocks %d: 1 or more, times page_size below 2^31", me, num_blocks);
    TLLM_REFUSE(kv_heads < 1 || kv_heads > kMaxHeads, "%s: kv_heads %d outside [1, %d]", me, kv_heads, kMaxHeads);
    TLLM_REFUSE(!pool || !aligned(pool, 16), "%s: the pool is null or not 16-byte aligned", me);
    TLLM_REFUSE(!scales || !aligned(scales, 4), "%s: the scales are null or not 4-byte aligned", me);
    return true;
}

bool append_fits(const tllm_paged_append_params_t* p)
{
    const char* const me = "tllm_paged_append";
    TLLM_REFUSE(!p, "%s: null parameters", me);
    TLLM_REFUSE(p->n_rows < 0 || p->n_rows > kMaxRows, "%s: n_rows %d outside [0, %d]", me, p->n_rows, kMaxRows);
    if (!cache_fits(me, p->dtype, p->cache_type, p->head_size, p->page_size, p->num_blocks, p->kv_heads, p->pool, p->scales))
        return false;
    TLLM_REFUSE(p->q_heads < 0 || p->q_heads > kMaxHeads, "%s: q_heads %d outside [0, %d]", me, p->q_heads, kMaxHeads);
    TLLM_REFUSE(p->rot_dim < 0 || p->rot_dim > p->head_size || p->rot_dim % 16, "%s: rot_dim %d is no multiple of 16 up to head_size %d", me, p->rot_dim, p->head_size);
    TLLM_REFUSE(p->rope_pairs != 0 && p->rope_pairs != 1, "%s: rope_pairs %d is neither 0 nor 1", me, p->rope_pairs);
    TLLM_REFUSE(p->rot_dim && (p->rope_len < 1 || !p->rope || !aligned(p->rope, 16)), "%s: rotation needs a 16-byte aligned rope table", me);
    TLLM_REFUSE(p->q_heads && !p->rot_dim, "%s: queries are only rotated here, and rot_dim is 0", me);
    if (p->n_rows == 0)
        return true;
    TLLM_REFUSE(!p->slot_map || !aligned(p->slot_map, 4), "%s: the slot map is null or not 4-byte aligned", me);
    TLLM_REFUSE(p->rot_dim && (!p->positions || !aligned(p->positions, 4)), "%s: the positions are null or not 4-byte aligned", me);
    if (!rows_fit(me, "k", p->k, p->k_row, p->k_head) || !rows_fit(me, "v", p->v, p->v_row, p->v_head))
        return false;
    if (p->q_heads == 0)
        return true;
    if (!rows_fit(me, "q", p->q, p->q_row, p->q_head) || !rows_fit(me, "q_out", p->q_out, p->q_out_row, p->q_out_head))
        return false;
    const Rows out(p->q_out, p->n_rows, p->q_out_row, p->q_heads, p->q_out_head, p->head_size), q(p->q, p->n_rows, p->q_row, p->q_heads, p->q_head, p->head_size);
    TLLM_REFUSE(folded(out), "%s: two rows of q_out lie on one place", me);
    TLLM_REFUSE((!(out == q) && overlap(out, q)) || overlap(out, Rows(p->k, p->n_rows, p->k_row, p->kv_heads, p->k_head, p->head_size))
            || overlap(out, Rows(p->v, p->n_rows, p->v_row, p->kv_heads, p->v_head, p->head_size)),
        "%s: q_out lies across q, k or v", me);
    return true;
}

bool attention_fits(const tllm_paged_attention_params_t* p)
{
    const char* const me = "tllm_paged_attention";
    TLLM_REFUSE(!p, "%s: null parameters", me);
    TLLM_REFUSE(p->n_seqs < 1 || p->n_seqs > kPlanMaxSeqs, "%s: n_seqs %d outside [1, %d]", me, p->n_seqs, kPlanMaxSeqs);
    TLLM_REFUSE(p->n_rows < 0 || p->n_rows > kMaxRows, "%s: n_rows %d outside [0, %d]", me, p->n_rows, kMaxRows);
    if (!cache_fits(me, p->dtype, p->cache_type, p->head_size, p->page_size, p->num_blocks, p->kv_heads, p->pool, p->scales))
        return false;
    TLLM_REFUSE(p->q_heads < 1 || p->q_heads > kMaxHeads || p->q_heads % p->kv_heads, "%s: q_heads %d is no multiple of kv_heads %d up to %d", me, p->q_heads, p->kv_heads, kMaxHeads);
    TLLM_REFUSE(p->max_blocks < 1 || p->max_blocks > kMaxRows, "%s: max_blocks %d outside [1, %d]", me, p->max_blocks, kMaxRows);
    TLLM_REFUSE(p->table_stride < p->max_blocks, "%s: table_stride %lld is less than max_blocks %d", me, (long long) p->table_stride, p->max_blocks);
    TLLM_REFUSE(p->max_new < 1 || p->max_new > kMaxRows, "%s: max_new %d outside [1, %d]", me, p->max_new, kMaxRows);
    TLLM_REFUSE(p->max_kv < 0 || p->window < 0, "%s: a negative max_kv or window", me);
    TLLM_REFUSE(!(p->scale >= 0.f && p->scale < 1e30f), "%s: the scale is negative or not finite", me);
    TLLM_REFUSE(!p->block_table || !p->cu_tokens || !p->kv_lens || !aligned(p->block_table, 4) || !aligned(p->cu_tokens, 4) || !aligned(p->kv_lens, 4),
        "%s: tables and lengths are null or not 4-byte aligned", me);
    // what does not go into one launch: row tiles of every request and key head, as many as one request may have
    const int64_t rows = (int64_t) std::min(p->max_new, p->n_rows) * (p->q_heads / p->kv_heads), in_tile = p->head_size == 256 ? 64 : 128;
    TLLM_REFUSE((int64_t) p->n_seqs * p->kv_heads * ((rows + in_tile - 1) / in_tile) > kMaxTiles, "%s: %d requests of up to %d rows are more than one launch takes", me, p->n_seqs,
        p->max_new);
    if (p->n_rows == 0)
        return true;
    if (!rows_fit(me, "q", p->q, p->q_row, p->q_head) || !rows_fit(me, "out", p->out, p->out_row, p->out_head))
        return false;
    const Rows out(p->out, p->n_rows, p->out_row, p->q_heads, p->out_head, p->head_size), q(p->q, p->n_rows, p->q_row, p->q_heads, p->q_head, p->head_size);
    TLLM_REFUSE(folded(out), "%s: two rows of out lie on one place", me);
    TLLM_REFUSE(!(out == q) && overlap(out, q), "%s: out lies across q", me);
    return true;
}

bool matmul_fits(const tllm_group_matmul_params_t* p)
{
    const char* const me = "tllm_group_matmul";
    TLLM_REFUSE(!p, "%s: null parameters", me);
    TLLM_REFUSE(p->dtype != TLLM_HALF && p->dtype != TLLM_BF16, "%s: dtype %d is neither float16 nor bfloat16", me, p->dtype);
    TLLM_REFUSE(p->group != 32 && p->group != 64 && p->group != 128, "%s: group %d is none of 32, 64, 128", me, p->group);
    TLLM_REFUSE(p->rows < 0 || p->rows > kMaxRows, "%s: rows %d outside [0, %d]", me, p->rows, kMaxRows);
    TLLM_REFUSE(p->n < 1 || p->n > (1 << 24) || p->k < 32 || p->k > (1 << 24) || p->k % 32, "%s: n %d, k %d: n in [1, 2^24], k a multiple of 32 up to 2^24", me, p->n, p->k);
    TLLM_REFUSE(!p->packed || !aligned(p->packed, 16) || !p->scales || !aligned(p->scales, 16), "%s: weights or scales are null or not 16-byte aligned", me);
    TLLM_REFUSE(p->rows && (!p->x || !aligned(p->x, 16) || p->ldx % 8 || (p->rows > 1 && p->ldx < p->k)), "%s: x has to be 16-byte aligned with a row stride that is a multiple of 8, at least k", me);
    TLLM_REFUSE(p->rows && (!p->y || !aligned(p->y, 2) || (p->rows > 1 && p->ldy < p->n)), "%s: y is null, not 2-byte aligned or its row stride is less than n", me);
    if (p->rows)
    {
        const int64_t tiles = (p->n + 15) / 16, groups = (p->k + p->group - 1) / p->group;
        const Range y(p->y, (int64_t) p->n * 2, p->rows, p->ldy * 2);
        TLLM_REFUSE(overlap(y, Range(p->x, (int64_t) p->k * 2, p->rows, p->ldx * 2)), "%s: y lies where x does", me);
        TLLM_REFUSE(overlap(y, Range(p->packed, tiles * ((p->k + 127) / 128) * 1024)) || overlap(y, Range(p->scales, groups * tiles * 32)), "%s: y lies where the weights do", me);
    }
    return true;
}

template <typename F>
int32_t guarded(F f)
{
    try
    {
        return f() ? 1 : 0;
    }
    catch (const std::exception& e)
    {
        set_error("%s", e.what());
        return 1;
    }
}
} // namespace

extern "C" {

int32_t tllm_paged_plan(const tllm_paged_plan_params_t* p, tllm_stream_t stream)
{
    return guarded([&] { return !plan_fits(p) || launch_paged_plan(*p, reinterpret_cast<hipStream_t>(stream)); });
}

int32_t tllm_paged_append(const tllm_paged_append_params_t* p, tllm_stream_t stream)
{
    return guarded([&] { return !append_fits(p) || (p->n_rows && launch_paged_append(*p, reinterpret_cast<hipStream_t>(stream))); });
}

// what the kernels get: a window that no row can fill is none (and does not take positions out of range), no request has more rows than there are
static tllm_paged_attention_params_t as_launched(const tllm_paged_attention_params_t& p)
{
    tllm_paged_attention_params_t q = p;
    if (q.window >= (int64_t) q.max_blocks * q.page_size)
        q.window = 0;
    q.max_new = std::min(q.max_new, q.n_rows);
    return q;
}

int64_t tllm_paged_attention_workspace(const tllm_paged_attention_params_t* p)
{
    int64_t bytes = -1;
    if (guarded([&] {
            if (!attention_fits(p))
                return true;
            bytes = p->n_rows ? (int64_t) paged_attention_workspace(as_launched(*p)) : 0;
            return false;
        }))
        return -1;
    return bytes;
}

int32_t tllm_paged_attention(const tllm_paged_attention_params_t* p, void* workspace, tllm_stream_t stream)
{
    return guarded([&] {
        if (!attention_fits(p))
            return true;
        if (p->n_rows == 0)
            return false;
        const tllm_paged_attention_params_t q = as_launched(*p);
        if (paged_attention_workspace(q) && (!workspace || !aligned(workspace, 16)))
        {
            set_error("tllm_paged_attention: the workspace is null or not 16-byte aligned");
            return true;
        }
        return launch_paged_attention(q, workspace, reinterpret_cast<hipStream_t>(stream)) != 0;
    });
}

int32_t tllm_group_matmul(const tllm_group_matmul_params_t* p, tllm_stream_t stream)
{
    return guarded([&] { return !matmul_fits(p) || (p->rows && launch_group_matmul(*p, reinterpret_cast<hipStream_t>(stream))); });
}

} // extern "C"
