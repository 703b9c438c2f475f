// attention.cpp -- C ABI of the row, prompt and 4-bit-cache attention kernels
// (include/smoe_hip.h): checks of what the host sees, plans, scratch, launches.
#include <cmath>
#include <initializer_list>
#include <utility>

#include "attention.hpp"
#include "context.hpp"

namespace {

constexpr uint64_t kMostRows = 1ull << 31;      // rows times heads of a call
// a launch has less than 2^32 threads: of the row kernels a wave a row or less, or 8192 in all
constexpr uint64_t kMostRowWaves = (1ull << 26) - 4;
constexpr uint64_t kMostStride = 1ull << 22;    // elements between rows
constexpr uint32_t kMostHeads = 1024;
constexpr uint32_t kMostPositions = 1u << 24;   // of a cache slot

bool bad_type(uint32_t t) { return t != SMOE_TYPE_F32 && t != SMOE_TYPE_F16 && t != SMOE_TYPE_BF16; }
bool bad_head_dim(uint32_t d) { return d != 64 && d != 128 && d != 256; }
uint32_t type_bytes(uint32_t t) { return t == SMOE_TYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// rows of `cols` elements, `stride` apart, in 16-byte pieces; nullptr if they can be had
const char* bad_rows(const void* p, uint64_t stride, uint64_t cols, uint32_t type)
{
    if (misaligned(p, 16)) return "rows are not 16-byte aligned";
    if (stride < cols) return "a row stride is less than its heads";
    if (stride * type_bytes(type) % 16) return "a row stride is no multiple of 16 bytes";
    if (stride > kMostStride) return "a row stride is over 2^22 elements";
    return nullptr;
}

// the context's device for the time of a call
class OnDevice {
public:
    explicit OnDevice(int device)
    {
        if (hipGetDevice(&before_) != hipSuccess || before_ == device) before_ = -1;
        else ok_ = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice()
    {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    bool ok() const { return ok_; }

private:
    int before_ = -1;
    bool ok_ = true;
};

template <typename A>
struct Launch {
    const A* a;
    uint32_t head_dim, type;
    hipStream_t stream;
    hipError_t (*f)(const A&, uint32_t, uint32_t, hipStream_t);
    static hipError_t run(void* p)
    {
        const Launch& l = *static_cast<Launch*>(p);
        return l.f(*l.a, l.head_dim, l.type, l.stream);
    }
};
template <typename A>
int launch(SmoeMetalCtx* ctx, uint32_t kind, const char* what, hipStream_t s,
           hipError_t (*f)(const A&, uint32_t, uint32_t, hipStream_t), const A& a, uint32_t head_dim, uint32_t type)
{
    Launch<A> l{&a, head_dim, type, s, f};
    return smoe::context_launch(ctx, kind, what, Launch<A>::run, &l);
}

int refuse(SmoeMetalCtx* ctx, int rc, const char* why) { return smoe::context_refuse(ctx, rc, why); }

// the cache's own fields
int check_cache(SmoeMetalCtx* ctx, const SmoeKv4Cache* c)
{
    if (!c->k_codes || !c->v_codes || !c->k_params || !c->v_params || c->n_slots == 0 || c->capacity == 0 ||
        c->num_kv_heads == 0)
        return refuse(ctx, SMOE_ERR_ARG, "a NULL or empty cache");
    if (bad_head_dim(c->head_dim)) return refuse(ctx, SMOE_ERR_SHAPE, "head_dim is not 64, 128 or 256");
    if (c->num_kv_heads > kMostHeads) return refuse(ctx, SMOE_ERR_SHAPE, "more than 1024 heads");
    // (a slot's codes of one head are addressed in 32 bits)
    if (c->n_slots > 0x7FFFFFFFu || c->capacity > kMostPositions)
        return refuse(ctx, SMOE_ERR_SHAPE, "more than 2^31 slots or 2^24 positions");
    if (misaligned(c->k_codes, 16) || misaligned(c->v_codes, 16) || misaligned(c->k_params, 16) ||
        misaligned(c->v_params, 16))
        return refuse(ctx, SMOE_ERR_ARG, "a cache buffer is not 16-byte aligned");
    return SMOE_OK;
}
smoe::Kv4 cache_of(const SmoeKv4Cache* c)
{
    return {{c->k_codes, c->v_codes}, {c->k_params, c->v_params}, c->n_slots, c->capacity, c->num_kv_heads};
}

int check_kv4_rows(SmoeMetalCtx* ctx, const SmoeKv4Cache* c, const SmoeKv4RowsArgs* a)
{
    if (!c || !a) return refuse(ctx, SMOE_ERR_ARG, "NULL arguments");
    if (const int rc = check_cache(ctx, c)) return rc;
    if (!a->k || !a->v || !a->start || a->n_seqs == 0) return refuse(ctx, SMOE_ERR_ARG, "NULL rows or start, or no sequence");
    if (bad_type(a->type)) return refuse(ctx, SMOE_ERR_ARG, "an unknown element type");
    if (!a->offsets && a->n_rows != a->n_seqs)
        return refuse(ctx, SMOE_ERR_ARG, "without offsets every sequence has one row");
    const uint64_t cols = uint64_t(c->num_kv_heads) * c->head_dim;
    for (const auto& r : {std::pair<const void*, uint64_t>(a->k, a->k_stride), {a->v, a->v_stride}})
        if (const char* why = bad_rows(r.first, r.second, cols, a->type)) return refuse(ctx, SMOE_ERR_SHAPE, why);
    // (a row's groups of 64 are dealt to waves in 32 bits)
    if (uint64_t(a->n_rows) * 2 * c->num_kv_heads * (c->head_dim / 64) >= kMostRows || a->n_rows > kMostRowWaves ||
        a->n_seqs >= kMostRows)
        return refuse(ctx, SMOE_ERR_SHAPE, "too many rows");
    return SMOE_OK;
}
smoe::Kv4Rows rows_of(const SmoeKv4Cache* c, const SmoeKv4RowsArgs* a, uint32_t* err)
{
    smoe::Kv4Rows r{};
    r.c = cache_of(c);
    r.rows[0] = a->k;
    r.rows[1] = a->v;
    r.stride[0] = a->k_stride;
    r.stride[1] = a->v_stride;
    r.offsets = a->offsets;
    r.slots = a->slots;
    r.start = a->start;
    r.n_seqs = a->n_seqs;
    r.n_rows = a->n_rows;
    r.err = err;
    return r;
}

}  // namespace

extern "C" int smoe_hip_qk_norm_rope(SmoeMetalCtx* ctx, const SmoeQkRowsArgs* a)
{
    if (!ctx) return SMOE_ERR_ARG;
    if (!a) return refuse(ctx, SMOE_ERR_ARG, "NULL arguments");
    if ((!a->q && !a->k) || !a->q != !a->q_out || !a->k != !a->k_out)
        return refuse(ctx, SMOE_ERR_ARG, "no rows, or rows without an output");
    if (!a->rope_cos != !a->rope_sin || (a->rope_cos && (!a->positions || a->n_positions == 0)))
        return refuse(ctx, SMOE_ERR_ARG, "RoPE needs both tables and the rows' positions");
    if (bad_type(a->type)) return refuse(ctx, SMOE_ERR_ARG, "an unknown element type");
    if (bad_head_dim(a->head_dim)) return refuse(ctx, SMOE_ERR_SHAPE, "head_dim is not 64, 128 or 256");
    if ((a->q && a->num_heads == 0) || (a->k && a->num_kv_heads == 0)) return refuse(ctx, SMOE_ERR_ARG, "rows of no heads");
    if (a->num_heads > kMostHeads || a->num_kv_heads > kMostHeads)
        return refuse(ctx, SMOE_ERR_SHAPE, "more than 1024 heads");
    if (misaligned(a->rope_cos, 16) || misaligned(a->rope_sin, 16) || misaligned(a->q_norm_w, 16) ||
        misaligned(a->k_norm_w, 16))
        return refuse(ctx, SMOE_ERR_ARG, "a table or norm weights are not 16-byte aligned");
    smoe::QkRows r{};
    if (a->q) {
        const uint64_t cols = uint64_t(a->num_heads) * a->head_dim;
        const char* why = bad_rows(a->q, a->q_stride, cols, a->type);
        if (!why) why = bad_rows(a->q_out, a->q_out_stride, cols, a->type);
        if (why) return refuse(ctx, SMOE_ERR_SHAPE, why);
        r.num_heads = a->num_heads;
    }
    if (a->k) {
        const uint64_t cols = uint64_t(a->num_kv_heads) * a->head_dim;
        const char* why = bad_rows(a->k, a->k_stride, cols, a->type);
        if (!why) why = bad_rows(a->k_out, a->k_out_stride, cols, a->type);
        if (why) return refuse(ctx, SMOE_ERR_SHAPE, why);
        r.num_kv_heads = a->num_kv_heads;
    }
    if (uint64_t(a->n_rows) * (r.num_heads + r.num_kv_heads) >= kMostRows || a->n_rows > kMostRowWaves)
        return refuse(ctx, SMOE_ERR_SHAPE, "too many rows");
    if (a->n_rows == 0) return SMOE_OK;
    const smoe::ContextView v = smoe::context_view(ctx);
    const OnDevice on(v.device);
    if (!on.ok()) return refuse(ctx, SMOE_ERR_HIP, "hipSetDevice failed");
    r.q = a->q;
    r.q_out = a->q_out;
    r.k = a->k;
    r.k_out = a->k_out;
    r.q_norm_w = a->q_norm_w;
    r.k_norm_w = a->k_norm_w;
    r.rope_cos = a->rope_cos;
    r.rope_sin = a->rope_sin;
    r.positions = a->positions;
    r.q_stride = a->q_stride;
    r.q_out_stride = a->q_out_stride;
    r.k_stride = a->k_stride;
    r.k_out_stride = a->k_out_stride;
    r.n_rows = a->n_rows;
    r.n_positions = a->n_positions;
    r.err = v.err;
    return launch(ctx, SMOE_KERNEL_QK_ROWS, "qk_norm_rope", v.stream, smoe::launch_qk_rows, r, a->head_dim, a->type);
}

extern "C" int smoe_hip_attention_prompt(SmoeMetalCtx* ctx, const SmoePromptAttnArgs* a)
{
    if (!ctx) return SMOE_ERR_ARG;
    if (!a) return refuse(ctx, SMOE_ERR_ARG, "NULL arguments");
    if (a->n_seqs == 0) return refuse(ctx, SMOE_ERR_ARG, "no sequence");
    if (!a->q_offsets || (a->q_rows && (!a->q || !a->out)) || (a->k_rows && (!a->k || !a->v)))
        return refuse(ctx, SMOE_ERR_ARG, "NULL rows or offsets");
    if (bad_type(a->type)) return refuse(ctx, SMOE_ERR_ARG, "an unknown element type");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return refuse(ctx, SMOE_ERR_ARG, "scale is not a positive number");
    if (bad_head_dim(a->head_dim)) return refuse(ctx, SMOE_ERR_SHAPE, "head_dim is not 64, 128 or 256");
    if (a->num_kv_heads == 0 || a->num_heads == 0 || a->num_heads % a->num_kv_heads)
        return refuse(ctx, SMOE_ERR_SHAPE, "num_heads is no multiple of num_kv_heads");
    if (a->num_heads > kMostHeads) return refuse(ctx, SMOE_ERR_SHAPE, "more than 1024 heads");
    const uint64_t qc = uint64_t(a->num_heads) * a->head_dim, kc = uint64_t(a->num_kv_heads) * a->head_dim;
    if (a->q_rows)
        for (const auto& r : {std::pair<const void*, uint64_t>(a->q, a->q_stride), {a->out, a->out_stride}})
            if (const char* why = bad_rows(r.first, r.second, qc, a->type)) return refuse(ctx, SMOE_ERR_SHAPE, why);
    if (a->k_rows)
        for (const auto& r : {std::pair<const void*, uint64_t>(a->k, a->k_stride), {a->v, a->v_stride}})
            if (const char* why = bad_rows(r.first, r.second, kc, a->type)) return refuse(ctx, SMOE_ERR_SHAPE, why);
    // (threads of a launch: 4 a row and head and 512 a sequence and KV head, or 8 a f32 key row and 256 a sequence)
    if (uint64_t(a->q_rows) * a->num_heads >= kMostRows / 4 || (uint64_t(a->n_seqs) + 8) * a->num_kv_heads >= 1u << 21 ||
        a->k_rows >= (a->type == SMOE_TYPE_F32 ? kMostRows / 8 : kMostRows))
        return refuse(ctx, SMOE_ERR_SHAPE, "too many rows or sequences");
    if (a->q_rows == 0) return SMOE_OK;
    const smoe::ContextView v = smoe::context_view(ctx);
    const OnDevice on(v.device);
    if (!on.ok()) return refuse(ctx, SMOE_ERR_HIP, "hipSetDevice failed");
    smoe::PromptAttn p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.out = a->out;
    p.q_offsets = a->q_offsets;
    p.k_offsets = a->k_offsets ? a->k_offsets : a->q_offsets;
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.out_stride = a->out_stride;
    p.n_seqs = a->n_seqs;
    p.q_rows = a->q_rows;
    p.k_rows = a->k_rows;
    p.num_kv_heads = a->num_kv_heads;
    p.group = a->num_heads / a->num_kv_heads;
    p.scale_log2 = a->scale * 1.44269504088896341f;
    p.err = v.err;
    smoe::prompt_plan(p, a->head_dim, a->type, a->max_k ? a->max_k : a->k_rows);
    if (const size_t need = smoe::prompt_scratch_bytes(p, a->head_dim)) {
        float* scratch = nullptr;
        if (const int rc = smoe::context_attention_scratch(ctx, need, &scratch)) return rc;
        smoe::prompt_scratch(p, a->head_dim, scratch);
    }
    return launch(ctx, SMOE_KERNEL_ATTENTION_PROMPT, "attention_prompt", v.stream, smoe::launch_attention_prompt, p,
                  a->head_dim, a->type);
}

extern "C" int smoe_hip_kv4_append(SmoeMetalCtx* ctx, const SmoeKv4Cache* c, const SmoeKv4RowsArgs* a)
{
    if (!ctx) return SMOE_ERR_ARG;
    if (const int rc = check_kv4_rows(ctx, c, a)) return rc;
    // other blocks still read these when the first one writes the lengths
    auto overlaps = [&](const int32_t* p, uint64_t n) {
        return a->lens_out && p && a->lens_out < p + n && p < a->lens_out + a->n_seqs;
    };
    if (overlaps(a->start, a->n_seqs) || overlaps(a->slots, a->n_seqs) || overlaps(a->offsets, uint64_t(a->n_seqs) + 1))
        return refuse(ctx, SMOE_ERR_ARG, "lens_out overlaps start, slots or offsets");
    const smoe::ContextView v = smoe::context_view(ctx);
    const OnDevice on(v.device);
    if (!on.ok()) return refuse(ctx, SMOE_ERR_HIP, "hipSetDevice failed");
    smoe::Kv4Rows r = rows_of(c, a, v.err);
    r.lens_out = a->lens_out;
    if (a->n_rows == 0 && !a->lens_out) return SMOE_OK;
    return launch(ctx, SMOE_KERNEL_KV4_ROWS, "kv4_append", v.stream, smoe::launch_kv4_append, r, c->head_dim, a->type);
}

extern "C" int smoe_hip_kv4_read(SmoeMetalCtx* ctx, const SmoeKv4Cache* c, const SmoeKv4RowsArgs* a)
{
    if (!ctx) return SMOE_ERR_ARG;
    if (const int rc = check_kv4_rows(ctx, c, a)) return rc;
    if (a->lens_out) return refuse(ctx, SMOE_ERR_ARG, "lens_out of a read");
    if (a->n_rows == 0) return SMOE_OK;
    const smoe::ContextView v = smoe::context_view(ctx);
    const OnDevice on(v.device);
    if (!on.ok()) return refuse(ctx, SMOE_ERR_HIP, "hipSetDevice failed");
    const smoe::Kv4Rows r = rows_of(c, a, v.err);
    return launch(ctx, SMOE_KERNEL_KV4_ROWS, "kv4_read", v.stream, smoe::launch_kv4_read, r, c->head_dim, a->type);
}

extern "C" int smoe_hip_attention_kv4(SmoeMetalCtx* ctx, const SmoeKv4Cache* c, const SmoeKv4AttnArgs* a)
{
    if (!ctx) return SMOE_ERR_ARG;
    if (!c || !a) return refuse(ctx, SMOE_ERR_ARG, "NULL arguments");
    if (const int rc = check_cache(ctx, c)) return rc;
    if (!a->q || !a->out || !a->lens || a->n_seqs == 0) return refuse(ctx, SMOE_ERR_ARG, "NULL rows or lens, or no sequence");
    if (bad_type(a->type)) return refuse(ctx, SMOE_ERR_ARG, "an unknown element type");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return refuse(ctx, SMOE_ERR_ARG, "scale is not a positive number");
    if (a->num_heads == 0 || a->num_heads % c->num_kv_heads)
        return refuse(ctx, SMOE_ERR_SHAPE, "num_heads is no multiple of num_kv_heads");
    if (a->num_heads > kMostHeads) return refuse(ctx, SMOE_ERR_SHAPE, "more than 1024 heads");
    const uint64_t cols = uint64_t(a->num_heads) * c->head_dim;
    for (const auto& r : {std::pair<const void*, uint64_t>(a->q, a->q_stride), {a->out, a->out_stride}})
        if (const char* why = bad_rows(r.first, r.second, cols, a->type)) return refuse(ctx, SMOE_ERR_SHAPE, why);
    // (256 threads a sequence and KV head, or 16 heads of it)
    if (uint64_t(a->n_seqs) * a->num_heads >= 1u << 24) return refuse(ctx, SMOE_ERR_SHAPE, "too many sequences");
    const smoe::ContextView v = smoe::context_view(ctx);
    const OnDevice on(v.device);
    if (!on.ok()) return refuse(ctx, SMOE_ERR_HIP, "hipSetDevice failed");
    smoe::Kv4Attn p{};
    p.c = cache_of(c);
    p.q = a->q;
    p.out = a->out;
    p.slots = a->slots;
    p.lens = a->lens;
    p.q_stride = a->q_stride;
    p.out_stride = a->out_stride;
    p.n_seqs = a->n_seqs;
    p.group = a->num_heads / c->num_kv_heads;
    p.scale_log2 = a->scale * 1.44269504088896341f;
    p.err = v.err;
    smoe::kv4_plan(p, c->head_dim, a->max_len ? a->max_len : c->capacity);
    if (const size_t need = smoe::kv4_scratch_bytes(p, c->head_dim))
        if (const int rc = smoe::context_attention_scratch(ctx, need, &p.part)) return rc;
    return launch(ctx, SMOE_KERNEL_ATTENTION_KV4, "attention_kv4", v.stream, smoe::launch_attention_kv4, p, c->head_dim,
                  a->type);
}
