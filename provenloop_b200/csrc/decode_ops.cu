// decode_ops.cu -- C entry points of the plaintext decode-step operators:
// checks of the arguments, the layout of the workspace, the device, and the
// launches.  Nothing here keeps state between calls.
#include <cstring>

#include "entry.cuh"
#include "lowrank.cuh"
#include "train.cuh"

using namespace tsg;

namespace {

constexpr uint64_t kMaxDim = 1u << 20, kMaxTokens = 1ull << 30;

int check_adapter(const ts_adapter_args* a, int backward) {
    if (!a) return bad("adapter arguments are NULL");
    if (a->dtype < TS_DTYPE_F32 || a->dtype > TS_DTYPE_F16) return bad("unknown dtype");
    if (a->d_in == 0 || a->d_in > kMaxDim || a->d_out == 0 || a->d_out > kMaxDim)
        return bad("d_in and d_out must be in 1 .. 2^20");
    if (a->r == 0 || a->r > TS_ADAPTER_MAX_RANK) return bad("the rank must be in 1 .. 256");
    if (a->adapters == 0 || a->adapters > 65535) return bad("the number of adapters must be in 1 .. 65535");
    if (a->n > kMaxTokens) return bad("at most 2^30 tokens in a call");
    if (a->tokens_per_id == 0) return bad("tokens_per_id is 0");
    const size_t size = dtype_size(a->dtype);
    if (!stride_ok(a->x_stride) || !stride_ok(a->out_stride) || (a->weight && !stride_ok(a->weight_stride)) ||
        (!backward && a->base && !stride_ok(a->base_stride)) || (backward && !stride_ok(a->grad_stride)))
        return bad("a stride is negative or above 2^40");
    if (backward) {
        if (a->n && !a->out && !a->grad_a) return bad("no gradient is asked for");
        if (!a->grad_a != !a->grad_b) return bad("grad_a and grad_b come together");
        if (a->bias || a->base) return bad("bias and base have no place in the backward call");
    } else if (a->grad || a->grad_a || a->grad_b) {
        return bad("grad, grad_a and grad_b have no place in the forward call");
    }
    if (a->n && (!a->x || !a->lora_a || !a->lora_b || !a->adapter || (backward ? !a->grad : !a->out)))
        return bad("a required pointer is NULL");
    for (const void* p : {a->x, a->weight, a->bias, a->base, a->lora_a, a->lora_b, a->grad, (const void*)a->out,
                          (const void*)a->grad_a, (const void*)a->grad_b})
        if (!aligned_to(p, size)) return bad("a pointer is not aligned to its type");
    if (!aligned_to(a->adapter, 4) || !aligned_to(a->scale, 4)) return bad("a pointer is not aligned to its type");
    const uint64_t ids = a->n ? (a->n - 1) / a->tokens_per_id + 1 : 0;
    const uint64_t wide = backward ? a->d_in : a->d_out;
    if (a->out && a->n > 1 && (uint64_t)a->out_stride < wide) return bad("rows of out overlap");
    const Region writes[] = {region(a->out, a->n, wide, a->out_stride, size),
                             region(a->grad_a, 1, (uint64_t)a->adapters * a->r * a->d_in, 0, size),
                             region(a->grad_b, 1, (uint64_t)a->adapters * a->r * a->d_out, 0, size),
                             region(a->workspace, 1, a->workspace_bytes, 0, 1)};
    const Region base = region(backward ? nullptr : a->base, a->n, a->d_out, a->base_stride, size);
    const Region reads[] = {region(a->x, a->n, a->d_in, a->x_stride, size),
                            region(a->weight, a->d_out, a->d_in, a->weight_stride, size),
                            region(a->bias, 1, a->d_out, 0, size),
                            region(a->lora_a, 1, (uint64_t)a->adapters * a->r * a->d_in, 0, size),
                            region(a->lora_b, 1, (uint64_t)a->adapters * a->r * a->d_out, 0, size),
                            region(a->grad, a->n, a->d_out, a->grad_stride, size),
                            region(a->adapter, 1, ids, 0, 4), region(a->scale, 1, a->adapters, 0, 4), base};
    for (const Region& w : writes) {
        for (const Region& r : reads) {
            const bool in_place = &w == writes && base.p && r.p == base.p && w.p == base.p && r.stride == w.stride && r.row == w.row &&
                                  &r == reads + sizeof(reads) / sizeof(reads[0]) - 1;
            if (!in_place && overlap(w, r)) return bad("what the call writes overlaps what it reads");
        }
        for (const Region& v : writes)
            if (&v != &w && overlap(w, v)) return bad("two results, or a result and the workspace, overlap");
    }
    return TS_OK;
}

// A row of `d` elements up to the next 16 bytes.
int up16(uint32_t d, size_t size) { return (int)((d * size + 15) / 16 * (16 / size)); }
int up8(uint32_t d) { return up16(d, 2); }

// Rows that 16-byte loads, bulk copies and TMA take as they are: on 16-byte
// boundaries, and one behind the other.
bool rows_ok(const void* p, uint64_t rows, uint32_t cols, int64_t stride, size_t size) {
    return aligned_to(p, 16) && (rows < 2 || (stride * size % 16 == 0 && stride >= cols && stride < (1ll << 38)));
}

// What a call does with its sizes and pointers, and where it puts it.
// Workspace: low (and for the backward call u); 16-bit operands whose rows are
// not on 16-byte boundaries are copied there first, as is the factor B of the
// backward call, transposed, so that its contraction axis is contiguous; the
// factor of the tensor-core projection in f32 with its flags; the tokens of
// each adapter.
struct Plan {
    bool f32, small, low_vec, out;
    bool pack_x, pack_w, pack_a, pack_grad, pack_b, g32, lists;
    uint64_t low, u, usplit, x, w, a, grad, b, g, bad, list, partial, bytes;
};

Plan plan_of(const ts_adapter_args* a, int backward) {
    Plan p{};
    p.f32 = a->dtype == TS_DTYPE_F32;
    p.out = !backward || a->out;
    const size_t size = dtype_size(a->dtype);
    const bool x_ok = rows_ok(a->x, a->n, a->d_in, a->x_stride, size), w_ok = rows_ok(a->weight, a->d_out, a->d_in, a->weight_stride, size);
    const bool a_ok = rows_ok(a->lora_a, 2, a->d_in, a->d_in, size), g_ok = rows_ok(a->grad, a->n, a->d_out, a->grad_stride, size);
    p.small = !p.f32 && !backward && a->n <= (uint64_t)kSmallTokens && (!a->weight || (x_ok && w_ok));
    const bool whole_low = !low_by_token((long long)a->n, a->d_in, a->d_in, a->r, a->adapters);  // by matrix instructions: aligned operands only
    if (p.f32) {
        p.low_vec = !backward && x_ok && a_ok;
        p.pack_x = backward && a->grad_a && !x_ok;
        p.pack_grad = backward && a->grad_a && !g_ok;
    } else if (!backward) {
        p.pack_x = !x_ok && ((a->weight && !p.small) || whole_low);
        p.pack_w = a->weight && !p.small && !w_ok;
        p.pack_a = !a_ok && whole_low;
        p.low_vec = (x_ok || p.pack_x) && (a_ok || p.pack_a);
        p.g32 = !p.small && !factor_by_token((long long)a->n, a->d_out, a->r, a->weight ? a->d_in : 0);
    } else {
        p.pack_x = !x_ok && a->grad_a;
        p.pack_a = !a_ok && a->grad_a;
        p.pack_w = a->weight && a->out && !w_ok;
        p.pack_grad = !g_ok;
        p.pack_b = true;
        p.low_vec = true;
        p.g32 = a->out && !factor_by_token((long long)a->n, a->d_in, a->r, a->weight ? a->d_out : 0);
    }
    p.lists = backward && a->grad_a;
    uint64_t at = 0;
    const auto take = [&](bool want, uint64_t bytes) {
        const uint64_t here = at;
        if (want) at += up(bytes);
        return here;
    };
    const uint64_t rs = low_stride((int)a->r), low = a->n * rs * 4, o = backward ? a->d_in : a->d_out;
    p.low = take(!backward || a->grad_a, low);
    p.u = take(backward, low);
    p.usplit = take(p.lists && a->dtype == TS_DTYPE_BF16, low);  // low itself is split then
    p.x = take(p.pack_x, a->n * up16(a->d_in, size) * size);
    p.w = take(p.pack_w, (uint64_t)a->d_out * up8(a->d_in) * 2);
    p.a = take(p.pack_a, (uint64_t)a->adapters * a->r * up8(a->d_in) * 2);
    p.grad = take(p.pack_grad, a->n * up16(a->d_out, size) * size);
    p.b = take(p.pack_b, (uint64_t)a->adapters * a->r * up8(a->d_out) * 2);
    p.g = take(p.g32, a->adapters * o * rs * 4);
    p.bad = take(p.g32, a->adapters * ((o + 127) / 128) * (rs / 16) * 4);
    p.list = take(p.lists, (a->adapters + 1 + a->n) * 4);
    p.partial = take(p.lists && a->n, a->n ? grad_partial_bytes((long long)a->n, a->d_in, a->d_out, (int)a->r, (int)a->adapters) : 0);
    p.bytes = a->n ? at : 0;
    return p;
}

AdapterIds ids_of(const ts_adapter_args* a) { return {a->adapter, (long long)a->tokens_per_id, (int)a->adapters}; }

int check_workspace(const ts_adapter_args* a, uint64_t need) {
    if (need && (!a->workspace || !aligned_to(a->workspace, 256) || a->workspace_bytes < need))
        return bad("the workspace is missing, not 256-byte aligned or smaller than ts_adapter_workspace says");
    return TS_OK;
}

int adapter_workspace(const ts_adapter_args* a, int backward, uint64_t* bytes) {
    if (!bytes) return bad("bytes is NULL");
    if (!a) return bad("adapter arguments are NULL");
    ts_adapter_args b = *a;
    b.workspace = nullptr;
    b.workspace_bytes = 0;
    const int rc = check_adapter(&b, backward);
    if (rc) return rc;
    *bytes = plan_of(a, backward).bytes;
    return TS_OK;
}

// Rows of a matrix or factor as the kernels take them: copied to the
// workspace first where `pack` is set.
struct Rows {
    const void* p;
    long long stride;
};

struct Work {
    const ts_adapter_args* a;
    cudaStream_t s;
    PackJobs jobs{};
    void* at(uint64_t off) const { return static_cast<char*>(a->workspace) + off; }
    Rows rows(bool pack, const void* p, uint64_t rows, uint32_t cols, long long stride, uint64_t off) {
        const size_t size = dtype_size(a->dtype);
        const int pitch = up16(cols, size), halves = (int)size / 2;  // elements are copied as 16-bit ones
        if (!pack) return {p, rows < 2 ? pitch : stride};
        jobs.add({PackJob::COPY, p, 0, stride * halves, 1, (long long)rows, 1, (int)cols * halves, pitch * halves, at(off)});
        return {at(off), pitch};
    }
    cudaError_t pack() {
        if (!jobs.jobs) return cudaSuccess;
        jobs.dtype = a->dtype;
        return launch_pack(jobs, s);
    }
};

int adapter_project(const ts_adapter_args* a) {
    int rc = check_adapter(a, 0);
    if (rc || a->n == 0) return rc;
    const Plan p = plan_of(a, 0);
    if ((rc = check_workspace(a, p.bytes))) return rc;
    OnDevice dev(a->device);
    if (dev.status != cudaSuccess) return cuda_status(dev.status);
    Work w{a, static_cast<cudaStream_t>(a->stream)};
    const long long n = (long long)a->n, rb = (long long)a->r * a->d_out;
    const int r = (int)a->r, d_o = (int)a->d_out;
    float* low = static_cast<float*>(w.at(p.low));
    const Rows x = p.f32 ? Rows{a->x, a->x_stride} : w.rows(p.pack_x, a->x, a->n, a->d_in, a->x_stride, p.x);
    const Rows wt = p.f32 ? Rows{a->weight, a->weight_stride} : w.rows(p.pack_w, a->weight, a->d_out, a->d_in, a->weight_stride, p.w);
    Rows fa{a->lora_a, a->d_in};
    if (p.pack_a) fa = w.rows(true, a->lora_a, (uint64_t)a->adapters * a->r, a->d_in, a->d_in, p.a);
    if (p.g32)
        w.jobs.add({PackJob::TO_F32, a->lora_b, rb, r, 1, d_o, (int)a->adapters, r, low_stride(r), w.at(p.g), static_cast<uint32_t*>(w.at(p.bad))});
    cudaError_t e = w.pack();
    const LowArgs l{x.p, x.stride, n, (int)a->d_in, r, {fa.p, r * fa.stride, fa.stride, 1}, ids_of(a), a->scale, low, nullptr, p.g32};
    const int after_pack = !w.jobs.jobs ? 0 : p.pack_x || p.pack_a ? 2 : 1;
    if (e == cudaSuccess) e = launch_low(&l, 1, a->dtype, p.low_vec, &after_pack, w.s);
    const ProjectArgs q{x.p, x.stride, n, (int)a->d_in, d_o, r, wt.p, wt.stride, 0, a->bias, a->base, a->base_stride, low, p.g32,
                        {a->lora_b, rb, 1, r}, p.g32 ? static_cast<float*>(w.at(p.g)) : nullptr, static_cast<uint32_t*>(w.at(p.bad)), ids_of(a), a->out, a->out_stride, p.pack_x || p.pack_w};
    if (e == cudaSuccess)
        e = p.f32 ? launch_project_f32(q, w.s) : p.small ? launch_project_small(q, a->dtype, w.s) : launch_project_tc(q, a->dtype, w.s);
    return cuda_status(e);
}

int adapter_project_backward(const ts_adapter_args* a) {
    int rc = check_adapter(a, 1);
    if (rc) return rc;
    const Plan p = plan_of(a, 1);
    if ((rc = check_workspace(a, p.bytes))) return rc;
    OnDevice dev(a->device);
    if (dev.status != cudaSuccess) return cuda_status(dev.status);
    Work w{a, static_cast<cudaStream_t>(a->stream)};
    const long long n = (long long)a->n, ra = (long long)a->r * a->d_in, rb = (long long)a->r * a->d_out;
    const int r = (int)a->r, di = (int)a->d_in, d_o = (int)a->d_out;
    if (n == 0) {
        if (!a->grad_a) return TS_OK;
        const size_t size = dtype_size(a->dtype);
        cudaError_t e = cudaMemsetAsync(a->grad_a, 0, (size_t)a->adapters * ra * size, w.s);
        if (e == cudaSuccess) e = cudaMemsetAsync(a->grad_b, 0, (size_t)a->adapters * rb * size, w.s);
        return cuda_status(e);
    }
    float *low = static_cast<float*>(w.at(p.low)), *u = static_cast<float*>(w.at(p.u));
    Rows x{a->x, a->x_stride}, wt{a->weight, a->weight_stride}, grad{a->grad, a->grad_stride}, fa{a->lora_a, di};
    Factor fb{a->lora_b, rb, 1, r};
    if (p.f32) {
        if (p.pack_x) x = w.rows(true, a->x, a->n, a->d_in, a->x_stride, p.x);
        if (p.pack_grad) grad = w.rows(true, a->grad, a->n, a->d_out, a->grad_stride, p.grad);
    } else {
        x = w.rows(p.pack_x, a->x, a->n, a->d_in, a->x_stride, p.x);
        wt = w.rows(p.pack_w, a->weight, a->d_out, a->d_in, a->weight_stride, p.w);
        grad = w.rows(p.pack_grad, a->grad, a->n, a->d_out, a->grad_stride, p.grad);
        if (p.pack_a) fa = w.rows(true, a->lora_a, (uint64_t)a->adapters * a->r, a->d_in, a->d_in, p.a);
        w.jobs.add({PackJob::COPY, a->lora_b, rb, 1, r, r, (int)a->adapters, d_o, up8(a->d_out), w.at(p.b)});
        fb = {w.at(p.b), (long long)r * up8(a->d_out), up8(a->d_out), 1};
    }
    if (p.g32)
        w.jobs.add({PackJob::TO_F32, a->lora_a, ra, 1, di, di, (int)a->adapters, r, low_stride(r), w.at(p.g), static_cast<uint32_t*>(w.at(p.bad))});
    int* first = static_cast<int*>(w.at(p.list));
    if (p.lists) {
        PackJob j{PackJob::LISTS};
        j.rows = n, j.count = (int)a->adapters, j.dst = first, j.id = ids_of(a);
        w.jobs.add(j);
    }
    cudaError_t e = w.pack();
    // u last: it needs the packed factor, low mostly nothing of the packing
    const bool split = a->dtype == TS_DTYPE_BF16 && a->grad_a;
    uint16_t* const lsplit = split ? reinterpret_cast<uint16_t*>(low) : nullptr;
    uint16_t* const usplit = split ? static_cast<uint16_t*>(w.at(p.usplit)) : nullptr;
    const int u_tf32 = p.g32 && (split || !a->grad_a);  // else the gradients read u too
    const LowArgs l[2] = {{x.p, x.stride, n, di, r, {fa.p, r * fa.stride, fa.stride, 1}, ids_of(a), a->scale, split ? nullptr : low, lsplit, 0},
                          {grad.p, grad.stride, n, d_o, r, fb, ids_of(a), a->scale, a->out || !split ? u : nullptr, usplit, u_tf32}};
    const int after_pack[2] = {!w.jobs.jobs ? 0 : p.pack_x || p.pack_a ? 2 : 1, !w.jobs.jobs ? 0 : p.pack_b || p.pack_grad ? 2 : 1};
    const int skip = a->grad_a ? 0 : 1;
    if (e == cudaSuccess) e = launch_low(l + skip, 2 - skip, a->dtype, p.low_vec, after_pack + skip, w.s);
    if (e == cudaSuccess && a->out) {
        const ProjectArgs q{grad.p, grad.stride, n, d_o, di, r, wt.p, wt.stride, 1, nullptr, nullptr, 0, u, u_tf32,
                            {a->lora_a, ra, di, 1}, p.g32 ? static_cast<float*>(w.at(p.g)) : nullptr, static_cast<uint32_t*>(w.at(p.bad)), ids_of(a), a->out, a->out_stride, p.pack_grad || p.pack_w};
        e = p.f32 ? launch_project_f32(q, w.s) : launch_project_tc(q, a->dtype, w.s);
    }
    if (e == cudaSuccess && a->grad_a) {
        const void *gu = split ? (const void*)usplit : u, *gl = split ? (const void*)lsplit : low;
        const GradPair g{{{x.p, x.stride, di, gu, a->grad_a, ra, di, 1}, {grad.p, grad.stride, d_o, gl, a->grad_b, rb, 1, r}},
                         r, (int)a->adapters, first, first + a->adapters + 1};
        e = launch_grads(g, n, a->dtype, !p.f32 && a->out, static_cast<float*>(w.at(p.partial)), w.s);
    }
    return cuda_status(e);
}

int logit_rules(const ts_rules_args* a) {
    if (!a) return bad("rules arguments are NULL");
    if (a->dtype < TS_DTYPE_F32 || a->dtype > TS_DTYPE_F16) return bad("unknown dtype");
    if (a->out && a->out_dtype != a->dtype && a->out_dtype != TS_DTYPE_F32) return bad("out_dtype must be dtype or f32");
    if (a->reserved) return bad("reserved must be 0");
    if (a->vocab == 0 || a->vocab > (1u << 30)) return bad("vocab must be in 1 .. 2^30");
    if (a->n > 1u << 27) return bad("at most 2^27 rows in a call");
    if (a->tokens && a->token_cols > TS_RULES_MAX_HISTORY) return bad("the history is longer than 1048575");
    if (a->bias_ids && a->bias_cols > TS_RULES_MAX_BIASES) return bad("more than 4095 biases in a row");
    if (!a->bias_ids != !a->bias_values) return bad("bias_ids and bias_values come together");
    if (!a->tokens && a->token_cols) return bad("the history is NULL");
    if (!stride_ok(a->logits_stride) || (a->out && !stride_ok(a->out_stride)) || (a->tokens && !stride_ok(a->tokens_stride)) ||
        (a->bias_ids && (!stride_ok(a->bias_ids_stride) || !stride_ok(a->bias_values_stride))) ||
        (a->mask && !stride_ok(a->mask_stride)))
        return bad("a stride is negative or above 2^40");
    if (a->n == 0) return TS_OK;
    if (!a->out && !a->pick) return bad("neither out nor pick is asked for");
    if (!a->logits) return bad("logits is NULL");
    const size_t size = dtype_size(a->dtype), osize = dtype_size(a->out_dtype);
    const size_t tsize = a->ids64 & 1 ? 8 : 4, bsize = a->ids64 & 2 ? 8 : 4;
    if (!aligned_to(a->logits, size) || !aligned_to(a->out, osize) || !aligned_to(a->tokens, tsize) || !aligned_to(a->bias_ids, bsize) ||
        !aligned_to(a->pick, 8))
        return bad("a pointer is not aligned to its type");
    for (const void* p : {(const void*)a->lengths, (const void*)a->prompt_lengths, (const void*)a->repetition, (const void*)a->frequency,
                          (const void*)a->presence, (const void*)a->bias_values, (const void*)a->mask})
        if (!aligned_to(p, 4)) return bad("a pointer is not aligned to its type");
    if (a->out && a->n > 1 && (uint64_t)a->out_stride < a->vocab) return bad("rows of out overlap");
    const Region logits = region(a->logits, a->n, a->vocab, a->logits_stride, size);
    const Region out = region(a->out, a->n, a->vocab, a->out_stride, osize), pick = region(a->pick, 1, a->n, 0, 8);
    const bool in_place = a->out == a->logits && a->dtype == a->out_dtype && a->out_stride == a->logits_stride;
    const Region reads[] = {region(a->tokens, a->n, a->token_cols, a->tokens_stride, tsize),
                            region(a->lengths, 1, a->n, 0, 4),
                            region(a->prompt_lengths, 1, a->n, 0, 4),
                            region(a->repetition, 1, a->n, 0, 4),
                            region(a->frequency, 1, a->n, 0, 4),
                            region(a->presence, 1, a->n, 0, 4),
                            region(a->bias_ids, a->n, a->bias_cols, a->bias_ids_stride, bsize),
                            region(a->bias_values, a->n, a->bias_cols, a->bias_values_stride, 4),
                            region(a->mask, a->n, (a->vocab + 31) / 32, a->mask_stride, 4)};
    for (const Region& r : reads)
        if (overlap(out, r) || overlap(pick, r)) return bad("what the call writes overlaps what it reads");
    if ((!in_place && overlap(out, logits)) || overlap(pick, logits) || overlap(out, pick))
        return bad("what the call writes overlaps what it reads");
    OnDevice dev(a->device);
    if (dev.status != cudaSuccess) return cuda_status(dev.status);
    const bool tokens = a->tokens && a->token_cols, biases = a->bias_ids && a->bias_cols;
    const RulesArgs k{a->logits, a->logits_stride, (long long)a->n, a->vocab,
                      tokens ? a->tokens : nullptr, a->tokens_stride, a->token_cols, a->ids64 & 1,
                      a->lengths, a->prompt_lengths, a->repetition, a->frequency, a->presence,
                      biases ? a->bias_ids : nullptr, a->bias_values, a->bias_ids_stride, a->bias_values_stride, a->bias_cols,
                      a->ids64 >> 1 & 1, reinterpret_cast<const uint32_t*>(a->mask), a->mask_stride, a->out, a->out_stride,
                      reinterpret_cast<long long*>(a->pick)};
    return cuda_status(launch_rules(k, a->dtype, a->out ? a->out_dtype : a->dtype, static_cast<cudaStream_t>(a->stream)));
}

}  // namespace

extern "C" int ts_adapter_workspace(const ts_adapter_args* args, int backward, uint64_t* bytes) {
    return guarded([&] { return adapter_workspace(args, backward, bytes); });
}
extern "C" int ts_adapter_project(const ts_adapter_args* args) {
    return guarded([&] { return adapter_project(args); });
}
extern "C" int ts_adapter_project_backward(const ts_adapter_args* args) {
    return guarded([&] { return adapter_project_backward(args); });
}
extern "C" int ts_expired_waits(int device, uint64_t* out) {
    if (!out) return bad("out is NULL");
    return guarded([&] {
        OnDevice dev(device);
        unsigned long long v = 0, w = 0, l = 0;
        cudaError_t e = dev.status;
        // the copies below wait for the legacy stream's work alone
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = expired_waits_project(&v);
        if (e == cudaSuccess) e = expired_waits_rules(&w);
        if (e == cudaSuccess) e = expired_waits_loss(&l);
        *out = v + w + l;
        return cuda_status(e);
    });
}
extern "C" int ts_logit_rules(const ts_rules_args* args) {
    return guarded([&] { return logit_rules(args); });
}
