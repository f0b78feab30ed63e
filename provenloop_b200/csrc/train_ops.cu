// train_ops.cu -- C entry points of the training operators: checks of the
// arguments, the layout of the workspace, the device, and the launches.
// Nothing here keeps state between calls.
#include <algorithm>
#include <cmath>
#include <vector>

#include "entry.cuh"
#include "train.cuh"

using namespace tsg;

namespace {

constexpr uint64_t kMaxRows = 1u << 27;

// What the call `op` reads and writes, apart from its workspace.
int check_loss(const ts_loss_args* a, int op) {
    if (!a) return bad("loss arguments are NULL");
    if (op < TS_LOSS_LOGPROBS || op > TS_LOSS_PREFERENCE) return bad("unknown call");
    if (a->dtype < TS_DTYPE_F32 || a->dtype > TS_DTYPE_F16) return bad("unknown dtype");
    if (a->vocab == 0 || a->vocab > (1u << 30)) return bad("vocab must be in 1 .. 2^30");
    if (a->n > kMaxRows) return bad("at most 2^27 rows in a call");
    if (a->reserved != 0.f) return bad("reserved must be 0");
    const bool back = op == TS_LOSS_LOGPROBS_BACKWARD, policy = op == TS_LOSS_POLICY, prefer = op == TS_LOSS_PREFERENCE;
    const bool loss = policy || prefer;
    if (!stride_ok(a->logits_stride) || (a->grad && !stride_ok(a->grad_stride))) return bad("a stride is negative or above 2^40");
    if (!loss && (a->sequences || a->starts || a->loss || a->margins || a->old_logprobs || a->ref_logprobs || a->advantages || a->grad_scale))
        return bad("arguments of the losses have no place in this call");
    if (!back && a->grad_logprobs) return bad("grad_logprobs has no place in this call");
    if (loss) {
        if (!a->loss) return bad("loss is NULL");
        if (a->sequences > (1u << 30)) return bad("at most 2^30 sequences in a call");
        if (!a->starts && (a->sequences ? a->n % a->sequences : a->n)) return bad("the rows do not divide into the sequences");
        if (a->starts && !a->sequences) return bad("starts needs sequences");
    }
    if (policy) {
        if (a->kind < TS_REDUCE_TOKEN || a->kind > TS_REDUCE_SUM) return bad("unknown reduction");
        if (!(a->clip_low >= 0.f) || !(a->clip_low <= 1.f) || !(a->clip_high >= 0.f)) return bad("clip_low must be in 0 .. 1 and clip_high not negative");
        if (!std::isfinite(a->kl)) return bad("kl must be finite");
        if (a->n && !a->advantages) return bad("advantages is NULL");
        if (a->margins) return bad("margins has no place in the policy loss");
    }
    if (prefer) {
        if (a->kind < TS_PREFER_SIGMOID || a->kind > TS_PREFER_SQUARED) return bad("unknown kind of preference loss");
        if (a->sequences % 2) return bad("the sequences are not pairs");
        if (!std::isfinite(a->beta) || !(a->beta > 0.f)) return bad("beta must be positive and finite");
        if (!(a->smoothing >= 0.f) || !(a->smoothing <= 0.5f)) return bad("smoothing must be in 0 .. 0.5");
        if (a->smoothing != 0.f && a->kind != TS_PREFER_SIGMOID) return bad("smoothing belongs to the sigmoid kind");
        if (a->old_logprobs || a->advantages) return bad("old_logprobs and advantages have no place in the preference loss");
    }
    const size_t size = dtype_size(a->dtype), tsize = a->targets64 ? 8 : 4;
    if (a->n && (!a->logits || !a->targets || (op == TS_LOSS_LOGPROBS && !a->logprobs) || (back && (!a->grad_logprobs || !a->grad))))
        return bad("a required pointer is NULL");
    if (back && a->logprobs) return bad("logprobs has no place in this call");
    if (op == TS_LOSS_LOGPROBS && a->grad) return bad("grad has no place in this call");
    if (!aligned_to(a->logits, size) || !aligned_to(a->grad, size) || !aligned_to(a->targets, tsize))
        return bad("a pointer is not aligned to its type");
    for (const void* p : {(const void*)a->grad_logprobs, (const void*)a->starts, (const void*)a->old_logprobs, (const void*)a->ref_logprobs,
                          (const void*)a->advantages, (const void*)a->grad_scale, (const void*)a->loss, (const void*)a->margins,
                          (const void*)a->logprobs})
        if (!aligned_to(p, 4)) return bad("a pointer is not aligned to its type");
    if (a->grad && a->n > 1 && (uint64_t)a->grad_stride < a->vocab) return bad("rows of grad overlap");
    const Region grad = region(a->grad, a->n, a->vocab, a->grad_stride, size), logits = region(a->logits, a->n, a->vocab, a->logits_stride, size);
    const Region writes[] = {grad, region(a->loss, 1, 1, 0, 4), region(a->margins, 1, a->sequences / 2, 0, 4),
                             region(a->logprobs, 1, a->n, 0, 4), region(a->workspace, 1, a->workspace_bytes, 0, 1)};
    const Region reads[] = {logits,
                            region(a->targets, 1, a->n, 0, tsize),
                            region(a->grad_logprobs, 1, a->n, 0, 4),
                            region(a->starts, 1, (uint64_t)a->sequences + 1, 0, 4),
                            region(a->old_logprobs, 1, a->n, 0, 4),
                            region(a->ref_logprobs, 1, a->n, 0, 4),
                            region(a->advantages, 1, a->advantage_rows ? a->n : a->sequences, 0, 4),
                            region(a->grad_scale, 1, 1, 0, 4)};
    const bool in_place = a->grad == a->logits && (a->grad_stride == a->logits_stride || a->n < 2);
    for (const Region& w : writes) {
        for (const Region& r : reads)
            if (!(in_place && &w == writes && &r == reads) && overlap(w, r)) return bad("what the call writes overlaps what it reads");
        for (const Region& v : writes)
            if (&v != &w && overlap(w, v)) return bad("two results, or a result and the workspace, overlap");
    }
    return TS_OK;
}

struct LossPlan {
    bool ordered;
    uint32_t tickets;
    uint64_t order, counts, stats, logs, slope, parts, ticket, bytes;
};

LossPlan plan_of(const ts_loss_args* a, int op) {
    LossPlan p{};
    uint64_t at = 0;
    const auto take = [&](bool want, uint64_t bytes) {
        const uint64_t here = at;
        if (want) at += up(bytes);
        return here;
    };
    const bool policy = op == TS_LOSS_POLICY, prefer = op == TS_LOSS_PREFERENCE;
    p.ordered = loss_orders(a->n, a->vocab, a->dtype, a->grad, prefer);
    p.order = take(p.ordered, (a->n + 1) * 4);
    p.counts = take(policy, ((uint64_t)a->sequences + 1) * 4);
    p.stats = take(prefer, a->n * sizeof(RowStats));
    p.logs = take(prefer, a->n * 8);
    p.slope = take(prefer, (uint64_t)a->sequences * 4);
    const uint64_t parts = policy ? a->n : a->sequences / 2;
    p.parts = take(policy || prefer, loss_sums(parts) * 8);
    p.tickets = (uint32_t)loss_tickets(parts);
    p.ticket = take(policy || prefer, p.tickets * 4ull);
    p.bytes = at;
    return p;
}

int loss_workspace(const ts_loss_args* a, int op, uint64_t* bytes) {
    if (!bytes) return bad("bytes is NULL");
    if (!a) return bad("loss arguments are NULL");
    ts_loss_args b = *a;
    b.workspace = nullptr;
    b.workspace_bytes = 0;
    const int rc = check_loss(&b, op);
    if (rc) return rc;
    *bytes = plan_of(a, op).bytes;
    return TS_OK;
}

int run_loss(const ts_loss_args* a, int op) {
    const int rc = check_loss(a, op);
    const bool loss = op == TS_LOSS_POLICY || op == TS_LOSS_PREFERENCE;
    if (rc || (!loss && a->n == 0)) return rc;
    const LossPlan p = plan_of(a, op);
    if (p.bytes && (!a->workspace || !aligned_to(a->workspace, 256) || a->workspace_bytes < p.bytes))
        return bad("the workspace is missing, not 256-byte aligned or smaller than ts_loss_workspace says");
    OnDevice dev(a->device);
    if (dev.status != cudaSuccess) return cuda_status(dev.status);
    const cudaStream_t s = static_cast<cudaStream_t>(a->stream);
    const LossRows r{a->logits, a->logits_stride, (long long)a->n, a->vocab, a->targets64, a->targets, a->sequences, a->starts,
                     (long long)(a->sequences ? a->n / a->sequences : 0)};
    const LossOut o{a->loss, a->margins, a->logprobs, a->grad, a->grad_stride, a->grad_scale};
    const auto at = [&](uint64_t off) { return static_cast<char*>(a->workspace) + off; };
    LossWork w{};
    if (p.ordered) w.order = reinterpret_cast<int*>(at(p.order));
    switch (op) {
        case TS_LOSS_LOGPROBS: return cuda_status(launch_logprobs(r, w, a->logprobs, a->dtype, s));
        case TS_LOSS_LOGPROBS_BACKWARD: return cuda_status(launch_logprobs_backward(r, a->grad_logprobs, w, o, a->dtype, s));
        case TS_LOSS_POLICY: {
            w.counts = reinterpret_cast<int*>(at(p.counts)), w.parts = reinterpret_cast<double*>(at(p.parts));
            w.ticket = reinterpret_cast<unsigned*>(at(p.ticket)), w.tickets = p.tickets;
            const PolicyTerms t{a->old_logprobs, a->ref_logprobs, a->advantages, a->advantage_rows, a->kind, 1.f - a->clip_low, 1.f + a->clip_high, a->kl};
            return cuda_status(launch_policy(r, t, w, o, a->dtype, s));
        }
        default: {
            if (!a->sequences) return cuda_status(cudaMemsetAsync(a->loss, 0, 4, s));
            w.stats = reinterpret_cast<RowStats*>(at(p.stats)), w.slope = reinterpret_cast<float*>(at(p.slope));
            w.logs = reinterpret_cast<double*>(at(p.logs)), w.parts = reinterpret_cast<double*>(at(p.parts));
            w.ticket = reinterpret_cast<unsigned*>(at(p.ticket)), w.tickets = p.tickets;
            const PreferTerms t{a->ref_logprobs, a->kind, a->average, a->beta, a->smoothing};
            return cuda_status(launch_preference(r, t, w, o, a->dtype, s));
        }
    }
}

constexpr uint64_t kMaxTensors = 1u << 20, kMaxElements = 1ull << 40;

// The checks of single arguments; the tensors that have elements.
int check_clip(const ts_clip_args* a, std::vector<ClipTensor>* parts) {
    if (!a) return bad("clip arguments are NULL");
    if (a->groups == 0 || a->groups > TS_CLIP_MAX_GROUPS) return bad("the number of groups must be in 1 .. 65535");
    if (a->count > kMaxTensors) return bad("at most 2^20 tensors in a call");
    if (a->count && !a->tensors) return bad("tensors is NULL");
    if (!a->norms) return bad("norms is NULL");
    if (!a->max_norms && !(a->max_norm >= 0.f)) return bad("max_norm must not be negative");
    if (!aligned_to(a->norms, 4) || !aligned_to(a->max_norms, 4)) return bad("a pointer is not aligned to its type");
    parts->reserve(a->count);
    uint64_t chunks = 0;
    for (uint64_t i = 0; i < a->count; i++) {
        const ts_clip_tensor& t = a->tensors[i];
        if (t.dtype < TS_DTYPE_F32 || t.dtype > TS_DTYPE_F16) return bad("unknown dtype");
        if (t.out_dtype != t.dtype && t.out_dtype != TS_DTYPE_F32) return bad("out_dtype must be dtype or f32");
        if (t.elements > kMaxElements) return bad("at most 2^40 elements in a tensor");
        if (a->groups > 1 && t.elements % a->groups) return bad("a tensor does not divide into the groups");
        if (t.elements == 0) continue;
        if (!t.grad || !t.out) return bad("a required pointer is NULL");
        if (!aligned_to(t.grad, dtype_size(t.dtype)) || !aligned_to(t.out, dtype_size(t.out_dtype))) return bad("a pointer is not aligned to its type");
        if (t.grad == t.out && t.dtype != t.out_dtype) return bad("a tensor and its result of another type overlap");
        parts->push_back({t.grad, t.out, t.elements / a->groups, t.dtype, t.out_dtype});
        chunks += (t.elements / a->groups + 4095) / 4096;
    }
    if (chunks * a->groups > 0x7fffffffull) return bad("the tensors are too many or too large for one call");
    return TS_OK;
}

// Nothing that is written may overlap anything else but a tensor its own
// result; tensors that are only read may overlap one another.
int check_clip_overlap(const ts_clip_args* a, const std::vector<ClipTensor>& parts) {
    struct Range {
        uintptr_t p, end;
        bool write;
    };
    std::vector<Range> all;
    all.reserve(2 * parts.size() + 3);
    const auto add = [&](const void* p, uint64_t bytes, bool write) {
        if (p && bytes) all.push_back({reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, write});
    };
    for (const ClipTensor& t : parts) {
        add(t.grad, t.part * a->groups * dtype_size(t.dtype), t.grad == t.out);
        if (t.grad != t.out) add(t.out, t.part * a->groups * dtype_size(t.out_dtype), true);
    }
    add(a->max_norms, a->one_max ? 4 : 4ull * a->groups, false);
    add(a->norms, 4ull * a->groups, true);
    add(a->workspace, a->workspace_bytes, true);
    // numbers of the ranges in the order of their starts: as one word each they sort three times as fast
    std::vector<uint64_t> order(all.size());
    const bool fits = all.size() < (1u << 17);
    for (size_t i = 0; i < all.size(); i++) order[i] = fits && !(all[i].p >> 47) ? (uint64_t)all[i].p << 17 | i : ~0ull;
    if (std::find(order.begin(), order.end(), ~0ull) == order.end()) {
        std::sort(order.begin(), order.end());
        for (uint64_t& o : order) o &= (1u << 17) - 1;
    } else {
        for (size_t i = 0; i < order.size(); i++) order[i] = i;
        std::sort(order.begin(), order.end(), [&](uint64_t x, uint64_t y) { return all[x].p < all[y].p; });
    }
    uintptr_t end = 0, write_end = 0;
    for (const uint64_t o : order) {
        const Range& r = all[o];
        if (r.p < write_end || (r.write && r.p < end)) return bad("tensors, results or the workspace overlap");
        end = std::max(end, r.end);
        if (r.write) write_end = std::max(write_end, r.end);
    }
    return TS_OK;
}

int clip_workspace(const ts_clip_args* a, uint64_t* bytes) {
    if (!bytes) return bad("bytes is NULL");
    if (!a) return bad("clip arguments are NULL");
    std::vector<ClipTensor> parts;
    const int rc = check_clip(a, &parts);
    if (rc) return rc;
    *bytes = clip_partials(parts.data(), parts.size(), a->groups) * 8;
    return TS_OK;
}

int clip_gradients(const ts_clip_args* a) {
    std::vector<ClipTensor> parts;
    int rc = check_clip(a, &parts);
    if (rc || (rc = check_clip_overlap(a, parts))) return rc;
    const uint64_t need = clip_partials(parts.data(), parts.size(), a->groups) * 8;
    if (!a->workspace || !aligned_to(a->workspace, 256) || a->workspace_bytes < need)
        return bad("the workspace is missing, not 256-byte aligned or smaller than ts_clip_workspace says");
    OnDevice dev(a->device);
    if (dev.status != cudaSuccess) return cuda_status(dev.status);
    const ClipArgs c{parts.data(), parts.size(), a->groups, a->max_norms, a->max_norm, a->one_max, a->norms, static_cast<double*>(a->workspace)};
    return cuda_status(launch_clip(c, static_cast<cudaStream_t>(a->stream)));
}

}  // namespace

extern "C" int ts_loss_workspace(const ts_loss_args* args, int op, uint64_t* bytes) {
    return guarded([&] { return loss_workspace(args, op, bytes); });
}
extern "C" int ts_token_logprobs(const ts_loss_args* args) {
    return guarded([&] { return run_loss(args, TS_LOSS_LOGPROBS); });
}
extern "C" int ts_token_logprobs_backward(const ts_loss_args* args) {
    return guarded([&] { return run_loss(args, TS_LOSS_LOGPROBS_BACKWARD); });
}
extern "C" int ts_policy_loss(const ts_loss_args* args) {
    return guarded([&] { return run_loss(args, TS_LOSS_POLICY); });
}
extern "C" int ts_preference_loss(const ts_loss_args* args) {
    return guarded([&] { return run_loss(args, TS_LOSS_PREFERENCE); });
}
extern "C" int ts_clip_workspace(const ts_clip_args* args, uint64_t* bytes) {
    return guarded([&] { return clip_workspace(args, bytes); });
}
extern "C" int ts_clip_gradients(const ts_clip_args* args) {
    return guarded([&] { return clip_gradients(args); });
}
