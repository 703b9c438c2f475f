// fake_attention.cpp -- launchers of the prompt and 4-bit-cache attention that only keep
// books, beside fake_hip.cpp, for the tests of csrc/attention.cpp on the CPU.
#include "attention.hpp"
#include "kernels.hpp"

#include <string.h>

#include <algorithm>

namespace {
uint64_t launches, splits, part;
hipError_t booked(uint32_t n_splits, const void* p)
{
    (void)smoe::dispatch_timer().take();
    if (n_splits > 1) (void)smoe::dispatch_timer().take();
    ++launches;
    splits = n_splits;
    part = reinterpret_cast<uint64_t>(p);
    return hipSuccess;
}
int device;
}  // namespace

extern "C" {
uint64_t fake_attention(const char* what)
{
    if (!strcmp(what, "launches")) return launches;
    if (!strcmp(what, "splits")) return splits;
    if (!strcmp(what, "device")) return static_cast<uint64_t>(device);
    return part;
}
hipError_t hipSetDevice(int d)
{
    device = d;
    return hipSuccess;
}
}

namespace smoe {
hipError_t launch_qk_rows(const QkRows&, uint32_t, uint32_t, hipStream_t) { return booked(1, nullptr); }
hipError_t launch_kv4_append(const Kv4Rows&, uint32_t, uint32_t, hipStream_t) { return booked(1, nullptr); }
hipError_t launch_kv4_read(const Kv4Rows&, uint32_t, uint32_t, hipStream_t) { return booked(1, nullptr); }
// plans of a simple rule: the entry points only pass them on
void prompt_plan(PromptAttn& a, uint32_t, uint32_t, uint32_t max_k) { a.splits = std::max(1u, std::min(64u, max_k / 256)); }
size_t prompt_scratch_bytes(const PromptAttn& a, uint32_t d)
{
    return a.splits == 1 ? 0 : 4 * part_floats(size_t(a.q_rows) * a.num_kv_heads * a.group, a.splits, d);
}
void prompt_scratch(PromptAttn& a, uint32_t, void* p) { a.part = static_cast<float*>(p); }
hipError_t launch_attention_prompt(const PromptAttn& a, uint32_t, uint32_t, hipStream_t) { return booked(a.splits, a.part); }
void kv4_plan(Kv4Attn& a, uint32_t, uint32_t max_len) { a.units = max_len < 512 ? 0 : a.n_seqs * std::min(64u, max_len / 256); }
size_t kv4_scratch_bytes(const Kv4Attn& a, uint32_t d)
{
    return a.units == 0 ? 0 : 4 * part_floats(size_t(a.units) * a.c.num_kv_heads * a.group, 1, d);
}
hipError_t launch_attention_kv4(const Kv4Attn& a, uint32_t, uint32_t, hipStream_t) { return booked(a.units ? 2 : 1, a.part); }
}  // namespace smoe
