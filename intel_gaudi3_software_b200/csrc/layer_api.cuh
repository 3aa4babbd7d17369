// C ABI of the 8-bit layer operators (mmeb200_rms_norm, mmeb200_rms_norm_grad, mmeb200_quantize, mmeb200_scaled_gemm):
// argument checks, staging, kernel choice. Part of api.cu's translation unit (it works on the context's internals).
#pragma once

namespace {

// The caller's current device is put back when the call returns.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before != device) cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int layer_elem_size(const mmeb200_tensor* t) { return t->dtype == MMEB200_INT8 ? 1 : dtype_size(t->dtype); }
bool layer_is_eight(int dtype) { return dtype == MMEB200_INT8 || dtype_is_fp8(dtype); }
bool layer_is_float(int dtype) { return dtype == DT_BF16 || dtype == DT_FP32; }

// The general rules of a tensor, with the data types a role accepts.
int layer_check(mmeb200_ctx* c, const mmeb200_tensor* t, const char* name, bool floats, bool eights) {
    if (!t) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: null tensor", name);
    if (t->dims < 1 || t->dims > 5) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: dims %d out of range", name, t->dims);
    if (!((floats && layer_is_float(t->dtype)) || (eights && layer_is_eight(t->dtype))))
        return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: data type %d is not accepted here", name, t->dtype);
    if (t->mem_space != MMEB200_MEM_HOST && t->mem_space != MMEB200_MEM_DEVICE) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: memory space %d is not valid", name, t->mem_space);
    if (t->strides[0] != 1) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: strides[0] must be 1", name);
    uint64_t n = 1;
    for (int d = 0; d < 5; ++d) {
        if (t->sizes[d] >= (1u << 31)) return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: tensors of 2^31 elements or more are not supported", name);
        n *= t->sizes[d];
        if (n >= (uint64_t(1) << 31)) return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: tensors of 2^31 elements or more are not supported", name);
    }
    if (n == 0) return 0;
    if (span_elems(t) >= (uint64_t(1) << 31)) return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: tensors of 2^31 elements or more are not supported", name);
    if (!t->data) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: null data", name);
    if (reinterpret_cast<uintptr_t>(t->data) % unsigned(layer_elem_size(t))) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: data is not aligned to its elements", name);
    return 0;
}
// Every element of an output has a place of its own.
int layer_check_distinct(mmeb200_ctx* c, const mmeb200_tensor* t, const char* name) {
    uint64_t reach = 1;   // elements spanned by the dims taken so far, in the order of their strides
    bool taken[5] = {};
    for (int k = 0; k < 5; ++k) {
        int best = -1;
        for (int d = 0; d < 5; ++d)
            if (!taken[d] && t->sizes[d] > 1 && (best < 0 || t->strides[d] < t->strides[best])) best = d;
        if (best < 0) break;
        taken[best] = true;
        if (t->strides[best] < reach) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: elements of an output overlap", name);
        reach += uint64_t(t->sizes[best] - 1) * t->strides[best];
    }
    return 0;
}
bool layer_same_place(const mmeb200_tensor* a, const mmeb200_tensor* b) {
    if (a->data != b->data || a->dtype != b->dtype) return false;
    for (int d = 0; d < 5; ++d)
        if (a->sizes[d] != b->sizes[d] || (a->sizes[d] > 1 && a->strides[d] != b->strides[d])) return false;
    return true;
}
// An output may share memory with an input only element by element (in_place), with another output never. Device tensors may lie
// between each other's rows; a host output is copied back with what lies between its rows, so there ranges count.
int layer_check_overlap(mmeb200_ctx* c, const mmeb200_tensor* out, const char* out_name, const mmeb200_tensor* other, const char* other_name, bool in_place) {
    if (!out || !other || out->mem_space != other->mem_space || num_elems(out) == 0 || num_elems(other) == 0) return 0;
    const uintptr_t a = reinterpret_cast<uintptr_t>(out->data), b = reinterpret_cast<uintptr_t>(other->data);
    if (a + span_elems(out) * layer_elem_size(out) <= b || b + span_elems(other) * layer_elem_size(other) <= a) return 0;
    if (in_place && layer_same_place(out, other)) return 0;
    if (out->mem_space == MMEB200_MEM_DEVICE) {
        uint64_t strides[8];
        for (int d = 1; d < 5; ++d) {
            strides[d - 1] = out->sizes[d] > 1 ? uint64_t(out->strides[d]) * layer_elem_size(out) : 0;
            strides[d + 3] = other->sizes[d] > 1 ? uint64_t(other->strides[d]) * layer_elem_size(other) : 0;
        }
        if (rows_lie_apart(a, uint64_t(out->sizes[0]) * layer_elem_size(out), b, uint64_t(other->sizes[0]) * layer_elem_size(other), strides)) return 0;
    }
    return c->fail(MMEB200_ERR_INVALID_ARG, "%s and %s overlap in memory", out_name, other_name);
}
int layer_same_sizes(mmeb200_ctx* c, const mmeb200_tensor* a, const mmeb200_tensor* b, const char* name) {
    for (int d = 0; d < 5; ++d)
        if (a->sizes[d] != b->sizes[d]) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: sizes do not match", name);
    return 0;
}
int layer_check_vector(mmeb200_ctx* c, const mmeb200_tensor* t, const char* name, uint64_t elems) {
    if (num_elems(t) != elems) return c->fail(MMEB200_ERR_INVALID_ARG, "%s: %llu elements, expected %llu", name, (unsigned long long) num_elems(t), (unsigned long long) elems);
    if (!is_dense(t)) return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: must be dense", name);
    return 0;
}
int layer_check_scale(mmeb200_ctx* c, const mmeb200_tensor* t, const char* name, uint64_t elems, bool one_for_all) {
    TRY(layer_check(c, t, name, true, false));
    if (t->dtype != DT_FP32) return c->fail(MMEB200_ERR_UNSUPPORTED, "%s: scales are fp32", name);
    return layer_check_vector(c, t, name, one_for_all && num_elems(t) == 1 ? 1 : elems);
}
// 0: not capturing, 1: capturing, or an error.
int layer_capturing(mmeb200_ctx* c, bool* capturing) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    CUDA_OK(c, cudaStreamIsCapturing(c->stream, &st));
    *capturing = st != cudaStreamCaptureStatusNone;
    return 0;
}
// Scratch memory of these operators. A captured call must not use it: a later call may replace it, and graphs that share it
// could run at the same time. Calls on different streams are ordered by the event that marks the last use.
int layer_scratch(mmeb200_ctx* c, size_t bytes, const char* remedy, void** out) {
    bool capturing = false;
    TRY(layer_capturing(c, &capturing));
    if (capturing) return c->fail(MMEB200_ERR_UNSUPPORTED, "this call needs scratch memory, which a captured call cannot use: %s", remedy);
    if (!c->layer_ws_used) CUDA_OK(c, cudaEventCreateWithFlags(&c->layer_ws_used, cudaEventDisableTiming));
    if (c->layer_ws_bytes < bytes) {
        CUDA_OK(c, cudaEventSynchronize(c->layer_ws_used));
        if (c->layer_ws) cudaFree(c->layer_ws);
        c->layer_ws = nullptr;
        c->layer_ws_bytes = 0;
        bytes = (bytes + (size_t(1) << 20) - 1) & ~((size_t(1) << 20) - 1);
        CUDA_OK(c, cudaMalloc(&c->layer_ws, bytes));
        c->layer_ws_bytes = bytes;
    }
    CUDA_OK(c, cudaStreamWaitEvent(c->stream, c->layer_ws_used, 0));
    *out = c->layer_ws;
    return 0;
}
// Records the event when the call that took scratch memory is through, or returns early.
struct LayerScratchMark {
    mmeb200_ctx* c;
    int operator()() const {
        CUDA_OK(c, cudaEventRecord(c->layer_ws_used, c->stream));
        return 0;
    }
};
using LayerScratchUse = UseMark<LayerScratchMark>;

// Host tensors are staged as everywhere else in this library; device tensors are used where they lie.
struct LayerStage {
    mmeb200_ctx* c;
    bool any_host = false;
    Staged staged[8];
    bool is_out[8] = {};
    int n = 0;
    explicit LayerStage(mmeb200_ctx* ctx) : c(ctx) {}
    int begin(std::initializer_list<const mmeb200_tensor*> all) {
        for (const mmeb200_tensor* t : all) any_host = any_host || (t && t->mem_space == MMEB200_MEM_HOST);
        if (!any_host) return 0;
        bool capturing = false;
        TRY(layer_capturing(c, &capturing));
        if (capturing) return c->fail(MMEB200_ERR_UNSUPPORTED, "a captured call takes device tensors only");
        arena_reset(c);
        return 0;
    }
    // *t points at the device image afterwards; nullptr stays nullptr. Gaps of a strided host output keep their contents.
    int add(const mmeb200_tensor** t, bool read, bool written) {
        if (!*t) return 0;
        Staged& s = staged[n];
        is_out[n] = written;
        ++n;
        TRY(stage_in(c, *t, &s, read || !is_dense(*t)));
        *t = &s.t;
        return 0;
    }
    int finish() {
        for (int i = 0; i < n; ++i)
            if (is_out[i]) TRY(stage_out(c, &staged[i]));
        return any_host ? collect_status(c) : 0;   // (every CUDA call's own status was looked at)
    }
};

int layer_row_type(int dtype) {
    return dtype == DT_BF16 ? ROW_BF16 : dtype == DT_FP32 ? ROW_F32 : dtype == MMEB200_INT8 ? ROW_I8 : ROW_F8;
}
RowTensor layer_rows(const mmeb200_tensor* t) {
    RowTensor r;
    memset(&r, 0, sizeof r);
    if (!t) return r;
    r.ptr = t->data;
    r.type = layer_row_type(t->dtype);
    for (int d = 0; d < 4; ++d) r.stride[d] = t->strides[d + 1];
    return r;
}
// Merges dims 1..4 into one where every tensor's strides allow it, so that a row's place needs no division.
void layer_flatten(uint32_t (&dims)[4], uint32_t* flat, std::initializer_list<RowTensor*> all) {
    int n = 0;
    for (int d = 1; d < 4; ++d) {
        if (dims[d] == 1) continue;
        bool merge = true;
        for (RowTensor* t : all)
            if (t->ptr && dims[n] != 1 && uint64_t(t->stride[n]) * dims[n] != t->stride[d]) merge = false;
        if (merge) {
            if (dims[n] == 1)
                for (RowTensor* t : all) t->stride[n] = t->stride[d];
            dims[n] *= dims[d];
        } else {
            ++n;
            dims[n] = dims[d];
            for (RowTensor* t : all) t->stride[n] = t->stride[d];
        }
    }
    for (int d = n + 1; d < 4; ++d) {
        dims[d] = 1;
        for (RowTensor* t : all) t->stride[d] = 0;
    }
    *flat = n == 0;
}
// How the rows of these tensors and gamma lie: 8, kPhased (where `phases` allows it) or 1 (norm_quant.h).
int layer_vector(uint32_t cols, const uint32_t (&dims)[4], std::initializer_list<const RowTensor*> all, const void* gamma, const void* partial, bool phases) {
    bool eight = cols % 8 == 0 && reinterpret_cast<uintptr_t>(partial) % 16 == 0;
    phases = phases && cols < (1u << 30);   // (phased columns are counted in 32 bits with a sign)
    const RowTensor* first = *all.begin();
    const auto elements = [](const RowTensor* t) { return reinterpret_cast<uintptr_t>(t->ptr) / (t->type >= ROW_I8 ? 1 : t->type == ROW_BF16 ? 2 : 4); };
    for (const RowTensor* t : all) {
        if (!t->ptr) continue;
        eight = eight && reinterpret_cast<uintptr_t>(t->ptr) % (t->type >= ROW_I8 ? 8 : 16) == 0;
        phases = phases && (elements(t) - elements(first)) % 8 == 0;
        for (int d = 0; d < 4; ++d) {
            if (dims[d] == 1) continue;
            eight = eight && t->stride[d] % 8 == 0;
            phases = phases && (t->stride[d] - first->stride[d]) % 8 == 0;
        }
    }
    if (reinterpret_cast<uintptr_t>(gamma) % 16 != 0) return 1;
    return eight ? 8 : phases ? kPhased : 1;
}
RowLaunch layer_launch(const mmeb200_ctx* c) { return RowLaunch{c->device, c->sm_count, c->stream, c->tune.dependent_launch != 0}; }

// Largest code of an 8-bit output and its hardware conversion.
int layer_codes(mmeb200_ctx* c, const mmeb200_tensor* out, float* top, Fp8HwCast* hw) {
    memset(hw, 0, sizeof *hw);
    *top = 127.0f;
    if (out->dtype == MMEB200_INT8) return 0;
    CastSpec s;
    mmeb200_cast_params cp;
    memset(&cp, 0, sizeof cp);
    cp.clip_fp = cp.clip_inf_in = 1;
    if (out->inf_nan_mode < 0 || out->inf_nan_mode > 2) return c->fail(MMEB200_ERR_INVALID_ARG, "output: Inf/NaN mode %d is not valid", out->inf_nan_mode);
    const bool e4m3 = out->dtype == DT_FP8_143;
    if (out->fp_bias < 1 || out->fp_bias > (e4m3 ? 15u : 30u)) return c->fail(MMEB200_ERR_INVALID_ARG, "output: exponent bias %u is out of range", out->fp_bias);
    TRY(make_cast_spec(c, out, &cp, &s));
    if (!cast_is_fp8_hw(s)) return c->fail(MMEB200_ERR_UNSUPPORTED, "output: 1-5-2 codes are written in the full Inf/NaN convention only");
    *hw = fp8_hw_cast(s);
    // largest finite value: 448 (minimal), 480 (no Inf / NaN), 240 (full) in 1-4-3 with bias 7, 57344 in 1-5-2 with bias 15
    const float base = !e4m3 ? 57344.0f : out->inf_nan_mode == 2 ? 448.0f : out->inf_nan_mode == 1 ? 480.0f : 240.0f;
    *top = ldexpf(base, (e4m3 ? 7 : 15) - int(out->fp_bias));
    return 0;
}

// Whether codes up to the type's largest finite value come from the hardware conversion alone (the 1-4-3 convention without
// infinities has codes above the hardware format's largest).
bool layer_direct(const mmeb200_tensor* out) { return dtype_is_fp8(out->dtype) && !(out->dtype == DT_FP8_143 && out->inf_nan_mode == MMEB200_INFNAN_NONE); }

// The scale argument of an 8-bit output, or its absence for a float output.
int layer_check_out_scale(mmeb200_ctx* c, const mmeb200_tensor* out, const mmeb200_tensor* scale, int scale_mode, uint64_t rows) {
    if (!layer_is_eight(out->dtype)) {
        if (scale) return c->fail(MMEB200_ERR_INVALID_ARG, "scale: a float output has none");
        return 0;
    }
    if (scale_mode != MMEB200_SCALE_ROW && scale_mode != MMEB200_SCALE_GIVEN) return c->fail(MMEB200_ERR_INVALID_ARG, "scale mode %d is not valid", scale_mode);
    return layer_check_scale(c, scale, "scale", rows, scale_mode == MMEB200_SCALE_GIVEN);
}

int run_rms_norm(mmeb200_ctx* c, mmeb200_tensor* out, mmeb200_tensor* scale, mmeb200_tensor* sum, const mmeb200_tensor* x, const mmeb200_tensor* residual,
                 const mmeb200_tensor* gamma, float eps, int scale_mode, bool norm) {
    TRY(layer_check(c, out, "output", norm, true));
    TRY(layer_check(c, x, "x", true, false));
    TRY(layer_same_sizes(c, out, x, "output"));
    if (residual) {
        TRY(layer_check(c, residual, "residual", true, false));
        TRY(layer_same_sizes(c, residual, x, "residual"));
    }
    if (sum) {
        if (!residual) return c->fail(MMEB200_ERR_INVALID_ARG, "sum: there is no residual to add");
        TRY(layer_check(c, sum, "sum", true, false));
        TRY(layer_same_sizes(c, sum, x, "sum"));
        if (sum->dtype != residual->dtype) return c->fail(MMEB200_ERR_INVALID_ARG, "sum: its data type is the residual's");
    }
    const uint64_t cols = x->sizes[0], rows = uint64_t(x->sizes[1]) * x->sizes[2] * x->sizes[3] * x->sizes[4];
    if (cols == 0) return c->fail(MMEB200_ERR_INVALID_ARG, "x: rows without elements");
    if (gamma) {
        TRY(layer_check(c, gamma, "gamma", true, false));
        TRY(layer_check_vector(c, gamma, "gamma", cols));
    }
    if (!(eps >= 0.0f) || std::isinf(eps)) return c->fail(MMEB200_ERR_INVALID_ARG, "eps must be finite and not negative");
    TRY(layer_check_out_scale(c, out, scale, scale_mode, rows));
    const bool eight = layer_is_eight(out->dtype), given = eight && scale_mode == MMEB200_SCALE_GIVEN;
    float top = 0.0f;
    Fp8HwCast hw;
    memset(&hw, 0, sizeof hw);
    if (eight) TRY(layer_codes(c, out, &top, &hw));
    TRY(layer_check_distinct(c, out, "output"));
    if (sum) TRY(layer_check_distinct(c, sum, "sum"));
    TRY(layer_check_overlap(c, out, "output", x, "x", true));
    TRY(layer_check_overlap(c, out, "output", residual, "residual", true));
    TRY(layer_check_overlap(c, out, "output", gamma, "gamma", false));
    TRY(layer_check_overlap(c, out, "output", sum, "sum", false));
    TRY(layer_check_overlap(c, out, "output", scale, "scale", false));
    TRY(layer_check_overlap(c, sum, "sum", x, "x", true));
    TRY(layer_check_overlap(c, sum, "sum", residual, "residual", true));
    TRY(layer_check_overlap(c, sum, "sum", gamma, "gamma", false));
    TRY(layer_check_overlap(c, sum, "sum", scale, "scale", false));
    if (!given) {
        TRY(layer_check_overlap(c, scale, "scale", x, "x", false));
        TRY(layer_check_overlap(c, scale, "scale", residual, "residual", false));
        TRY(layer_check_overlap(c, scale, "scale", gamma, "gamma", false));
    }
    if (rows == 0) return 0;
    LayerStage st(c);
    const mmeb200_tensor *dx = x, *dres = residual, *dgam = gamma, *dsum = sum, *dout = out, *dscale = scale;
    TRY(st.begin({x, residual, gamma, sum, out, scale}));
    TRY(st.add(&dx, true, false));
    TRY(st.add(&dres, true, false));
    TRY(st.add(&dgam, true, false));
    TRY(st.add(&dsum, false, true));
    TRY(st.add(&dout, false, true));
    TRY(st.add(&dscale, given, !given));
    NormParams p;
    memset(&p, 0, sizeof p);
    p.x = layer_rows(dx); p.residual = layer_rows(dres); p.sum = layer_rows(dsum); p.out = layer_rows(dout);
    p.gamma = layer_rows(dgam);
    if (dscale) {
        if (given) { p.given = static_cast<const float*>(dscale->data); p.given_stride = num_elems(dscale) == 1 ? 0 : 1; }
        else p.scale = static_cast<float*>(dscale->data);
    }
    p.rows = uint32_t(rows); p.cols = uint32_t(cols);
    for (int d = 0; d < 4; ++d) p.dims[d] = x->sizes[d + 1];
    layer_flatten(p.dims, &p.flat, {&p.x, &p.residual, &p.sum, &p.out});
    p.norm = norm; p.eps = eps; p.per_col = 1.0f / float(cols); p.top = top; p.hw = hw;
    p.fp8_direct = layer_direct(out);
    p.mode = out->dtype == DT_BF16 ? NORM_BF16 : out->dtype == DT_FP32 ? NORM_F32 : out->dtype == MMEB200_INT8 ? (given ? NORM_I8_GIVEN : NORM_I8) : given ? NORM_F8_GIVEN : NORM_F8;
    const int vec = layer_vector(p.cols, p.dims, {&p.x, &p.residual, &p.sum, &p.out}, p.gamma.ptr, nullptr, true);
    CUDA_OK(c, launch_norm(layer_launch(c), p, vec));
    c->launches++;
    return st.finish();
}

int run_rms_norm_grad(mmeb200_ctx* c, mmeb200_tensor* dx, mmeb200_tensor* dgamma, const mmeb200_tensor* dy, const mmeb200_tensor* x, const mmeb200_tensor* gamma,
                      const mmeb200_tensor* dsum, float eps, mmeb200_tensor* workspace) {
    TRY(layer_check(c, dx, "dx", true, false));
    TRY(layer_check(c, dy, "dy", true, false));
    TRY(layer_check(c, x, "x", true, false));
    TRY(layer_same_sizes(c, dx, x, "dx"));
    TRY(layer_same_sizes(c, dy, x, "dy"));
    if (dy->dtype != x->dtype || dx->dtype != x->dtype) return c->fail(MMEB200_ERR_UNSUPPORTED, "dx, dy and x have one data type");
    if (dsum) {
        TRY(layer_check(c, dsum, "dsum", true, false));
        TRY(layer_same_sizes(c, dsum, x, "dsum"));
        if (dsum->dtype != x->dtype) return c->fail(MMEB200_ERR_UNSUPPORTED, "dsum: its data type is x's");
    }
    const uint64_t cols = x->sizes[0], rows = uint64_t(x->sizes[1]) * x->sizes[2] * x->sizes[3] * x->sizes[4];
    if (cols == 0) return c->fail(MMEB200_ERR_INVALID_ARG, "x: rows without elements");
    if (gamma) {
        TRY(layer_check(c, gamma, "gamma", true, false));
        TRY(layer_check_vector(c, gamma, "gamma", cols));
    }
    if (dgamma) {
        TRY(layer_check(c, dgamma, "dgamma", true, false));
        if (dgamma->dtype != DT_FP32) return c->fail(MMEB200_ERR_UNSUPPORTED, "dgamma: the sum over rows is fp32");
        TRY(layer_check_vector(c, dgamma, "dgamma", cols));
    }
    if (!(eps >= 0.0f) || std::isinf(eps)) return c->fail(MMEB200_ERR_INVALID_ARG, "eps must be finite and not negative");
    uint32_t blocks = norm_grad_blocks(c->device, c->sm_count, uint32_t(rows), uint32_t(cols));
    const uint64_t need = uint64_t(blocks) * cols;
    if (workspace) {
        TRY(layer_check(c, workspace, "workspace", true, false));
        if (workspace->dtype != DT_FP32 || workspace->mem_space != MMEB200_MEM_DEVICE || !is_dense(workspace))
            return c->fail(MMEB200_ERR_UNSUPPORTED, "workspace: a dense fp32 device tensor");
        if (dgamma && num_elems(workspace) < need)
            return c->fail(MMEB200_ERR_INVALID_ARG, "workspace: %llu elements, %llu are needed", (unsigned long long) num_elems(workspace), (unsigned long long) need);
    }
    TRY(layer_check_distinct(c, dx, "dx"));
    TRY(layer_check_overlap(c, dx, "dx", x, "x", true));
    TRY(layer_check_overlap(c, dx, "dx", dy, "dy", true));
    TRY(layer_check_overlap(c, dx, "dx", dsum, "dsum", true));
    TRY(layer_check_overlap(c, dx, "dx", gamma, "gamma", false));
    TRY(layer_check_overlap(c, dx, "dx", dgamma, "dgamma", false));
    for (const mmeb200_tensor* t : {x, dy, dsum, gamma, (const mmeb200_tensor*) dx, (const mmeb200_tensor*) dgamma})
        if (workspace) TRY(layer_check_overlap(c, workspace, "workspace", t, "another tensor", false));
    if (dgamma)
        for (const mmeb200_tensor* t : {x, dy, dsum, gamma}) TRY(layer_check_overlap(c, dgamma, "dgamma", t, "an input", false));
    if (rows == 0 && !dgamma) return 0;
    LayerStage st(c);
    const mmeb200_tensor *tx = x, *ty = dy, *ts = dsum, *tg = gamma, *to = dx, *tdg = dgamma;
    TRY(st.begin({x, dy, dsum, gamma, dx, dgamma}));
    TRY(st.add(&tx, true, false));
    TRY(st.add(&ty, true, false));
    TRY(st.add(&ts, true, false));
    TRY(st.add(&tg, true, false));
    TRY(st.add(&to, false, true));
    TRY(st.add(&tdg, false, true));
    if (rows == 0) {   // an empty sum
        CUDA_OK(c, cudaMemsetAsync(tdg->data, 0, cols * sizeof(float), c->stream));
        return st.finish();
    }
    NormGradParams p;
    memset(&p, 0, sizeof p);
    p.x = layer_rows(tx); p.dy = layer_rows(ty); p.dsum = layer_rows(ts); p.dx = layer_rows(to);
    p.gamma = layer_rows(tg);
    p.rows = uint32_t(rows); p.cols = uint32_t(cols);
    for (int d = 0; d < 4; ++d) p.dims[d] = x->sizes[d + 1];
    layer_flatten(p.dims, &p.flat, {&p.x, &p.dy, &p.dsum, &p.dx});
    p.eps = eps; p.per_col = 1.0f / float(cols);
    LayerScratchUse use(LayerScratchMark{c});
    if (dgamma) {
        if (workspace) p.partial = static_cast<float*>(workspace->data);
        else {
            void* scratch = nullptr;
            TRY(layer_scratch(c, need * sizeof(float), "pass a workspace", &scratch));
            use.begin();
            p.partial = static_cast<float*>(scratch);
        }
    }
    const uint32_t phased = norm_grad_phased_blocks(blocks, p.rows, p.cols);
    const int vec = layer_vector(p.cols, p.dims, {&p.x, &p.dy, &p.dsum, &p.dx}, p.gamma.ptr, p.partial, p.flat && p.cols % 8 != 0 && phased > 0);
    if (vec == kPhased) blocks = phased;
    CUDA_OK(c, launch_norm_grad(layer_launch(c), p, vec, blocks));
    c->launches++;
    if (dgamma) {
        CUDA_OK(c, launch_column_sums(layer_launch(c), p.partial, static_cast<float*>(tdg->data), blocks, uint32_t(cols)));
        c->launches++;
    }
    TRY(use.end());
    return st.finish();
}

int run_quantize(mmeb200_ctx* c, mmeb200_tensor* out, mmeb200_tensor* scale, const mmeb200_tensor* x, int op, int scale_mode) {
    if (op != MMEB200_OP_MEMCPY && op != MMEB200_OP_TRANS) return c->fail(MMEB200_ERR_INVALID_ARG, "operation %d is neither MEMCPY nor TRANS", op);
    if (op == MMEB200_OP_MEMCPY) {
        if (!scale) return c->fail(MMEB200_ERR_INVALID_ARG, "scale: null tensor");
        return run_rms_norm(c, out, scale, nullptr, x, nullptr, nullptr, 0.0f, scale_mode, false);
    }
    TRY(layer_check(c, out, "output", false, true));
    TRY(layer_check(c, x, "x", true, false));
    for (int d = 2; d < 5; ++d)
        if (x->sizes[d] != 1 || out->sizes[d] != 1) return c->fail(MMEB200_ERR_UNSUPPORTED, "a transposed quantisation is 2-D");
    if (out->sizes[0] != x->sizes[1] || out->sizes[1] != x->sizes[0]) return c->fail(MMEB200_ERR_INVALID_ARG, "output: sizes are not x's transposed");
    const uint64_t cols = x->sizes[0], rows = x->sizes[1];
    if (rows == 0) return c->fail(MMEB200_ERR_INVALID_ARG, "x: columns without elements");
    TRY(layer_check_out_scale(c, out, scale, scale_mode, cols));
    const bool given = scale_mode == MMEB200_SCALE_GIVEN;
    QuantTransParams p;
    memset(&p, 0, sizeof p);
    TRY(layer_codes(c, out, &p.top, &p.hw));
    p.fp8_direct = layer_direct(out);
    TRY(layer_check_distinct(c, out, "output"));
    TRY(layer_check_overlap(c, out, "output", x, "x", false));
    TRY(layer_check_overlap(c, out, "output", scale, "scale", false));
    if (!given) TRY(layer_check_overlap(c, scale, "scale", x, "x", false));
    if (cols == 0) return 0;
    LayerStage st(c);
    const mmeb200_tensor *tx = x, *to = out, *ts = scale;
    TRY(st.begin({x, out, scale}));
    TRY(st.add(&tx, true, false));
    TRY(st.add(&to, false, true));
    TRY(st.add(&ts, given, !given));
    p.x = layer_rows(tx); p.x_ld = tx->strides[1];
    p.out = to->data; p.out_type = layer_row_type(to->dtype); p.out_ld = to->strides[1];
    if (given) { p.given = static_cast<const float*>(ts->data); p.given_stride = num_elems(ts) == 1 ? 0 : 1; }
    else p.scale = static_cast<float*>(ts->data);
    p.rows = uint32_t(rows); p.cols = uint32_t(cols);
    int launches = 0;
    const uint32_t dims[4] = {p.rows, 1, 1, 1};
    CUDA_OK(c, launch_quant_trans(layer_launch(c), p, layer_vector(p.cols, dims, {&p.x}, nullptr, nullptr, true), &launches));
    c->launches += uint64_t(launches);
    return st.finish();
}

// One operand of a scaled product: K-major rows for TMA, copied to 16-byte rows where they are not.
bool layer_operand(const mmeb200_tensor* t, TmaOperand* o) {
    o->ptr = t->data; o->elem = 1; o->mn_major = false;
    o->inner = t->sizes[0]; o->rows = t->sizes[1]; o->row_stride = t->strides[1];
    o->hw_fmt = t->dtype == DT_FP8_152 ? 1 : 0;
    // rows that share memory (a stride below their length) are read like any others
    return tma_compatible(*o) && (o->rows == 1 || o->row_stride != 0);
}
// Copies of a product's operands that have to be made before it. They are launched when nothing else of the call can fail but
// the product's own launch.
struct LayerPads {
    TmaOperand from[2], to[2];
    int n = 0;
    static uint64_t bytes(const TmaOperand& o) { return o.rows * ((o.inner + 15) & ~uint64_t(15)); }
    // *o lies at dst from now on
    void add(TmaOperand* o, uint8_t* dst) {
        from[n] = *o;
        o->ptr = dst;
        o->row_stride = (o->inner + 15) & ~uint64_t(15);
        to[n++] = *o;
    }
    int launch(mmeb200_ctx* c) const {
        for (int i = 0; i < n; ++i) {
            CUDA_OK(c, launch_pad_rows(layer_launch(c), from[i].ptr, const_cast<void*>(to[i].ptr), from[i].rows, from[i].inner, from[i].row_stride, to[i].row_stride));
            c->launches++;
        }
        return 0;
    }
};

int layer_token_capacity(mmeb200_ctx* c, uint32_t kind, uint32_t tok, uint32_t splits, uint32_t ctas) {
    static std::atomic<int> known[64][2][4][9] = {};   // of the full ring, which all tiles nearly have
    return device_holds(known[c->device & 63][kind == KIND_I8][ctas][splits], [&](int* n) { return gemm_tokens_capacity(launch_env(c), kind, tok, splits, ctas, n); },
                        [] { cudaGetLastError(); });
}
// Which kernel a product takes, and with what tile and split: the choice with the least estimated time, a function of the
// sizes alone. The estimates (microseconds) are sums of a few measured rates, which reproduce the measured times of some
// twenty shapes from 8 x 512 x 512 to 8192^3, both kernels forced in turn, mostly within 15 %:
//   few-token kernel: 2.5 to launch; then the larger of HBM's 6050 bytes/ns for what is read and written once and of what the
//     busiest SM takes in, 130 bytes/ns; then its epilogue, 25 ns per token of the tile, or the exchange of a split tile.
//     Two CTAs per SM hide one's epilogue behind the other's loads, but share an SM where the device has SMs to spare.
//   CTA-pair kernel: 0.355 per k block and wave of 256 x 256 tiles, or the epilogue where that takes longer.
// (int8 256 x 8192 x 8192: 20 us on the first, 36 us on the second; 512 x 8192 x 8192: 33 and 28 us.)
ProductPlan layer_make_plan(mmeb200_ctx* c, uint32_t kind, uint32_t M, uint32_t N, uint32_t kb, uint32_t out_bytes, bool rows_aligned) {
    const double sms = c->sm_count, hbm = (128.0 * kb * (double(M) + N) + double(M) * N * out_bytes) / 6.05e6;
    ProductPlan best{false, 0, 0, 0, 1e300};
    if (c->tune.pair != 0 && M >= 256 && N >= 256) {
        const double tiles = double((M + 255) / 256) * ((N + 255) / 256), waves = ceil(tiles / floor(sms / 2)), epilogue = rows_aligned ? 4.3 : 6.0;
        best = {true, 0, 0, 0, 3.0 + std::max(hbm, waves * std::max(kb * 0.355, epilogue)) + (rows_aligned ? 2.0 : epilogue)};
        if (c->tune.pair == 1) return best;
    }
    const double channels = double((uint64_t(N) + kBlockM - 1) / kBlockM);
    uint32_t before = 0;
    for (uint32_t want : {256u, 192u, 128u, 112u, 96u, 80u, 64u, 48u, 32u, 16u}) {
        if (c->tune.token_tile > 0) want = std::min(256u, (uint32_t(c->tune.token_tile) + 15) & ~15u);
        // the smallest tile with as many token tiles as tiles of `want` tokens would give
        const uint32_t m_tiles = (M + want - 1) / want, tok = c->tune.token_tile > 0 ? want : ((M + m_tiles - 1) / m_tiles + 15) & ~15u;
        const double stage = kBlockM * kRowBytes + tok * kRowBytes, tiles = channels * m_tiles;
        const double memory = hbm + 0.25 * (m_tiles - 1) * 128.0 * kb * N / 6.05e6;   // a quarter of the weights' further reads misses L2
        if (tok == before) continue;
        before = tok;
        for (uint32_t s = 1; s <= 8 && s <= kb; ++s) {
            const uint32_t per = (kb + s - 1) / s;
            if (per * (s - 1) >= kb) continue;   // no share may be empty
            if (c->tune.token_split > 0) {
                if (s != std::min(uint32_t(c->tune.token_split), 8u) && s != 1) continue;   // 1 where that many do not exist
            } else if (tiles * (s - 1) > 2 * sms) {
                break;   // more CTAs than the device takes at once gain nothing
            }
            const double ctas_all = tiles * s, epilogue = s == 1 ? 0.025 * tok : 0.9 + tok * (0.010 + 0.040 / s);
            const bool wanted = c->tune.token_split > 0 && s == std::min(uint32_t(c->tune.token_split), 8u);
            for (uint32_t ctas = 1; ctas <= 2; ++ctas) {
                if (gemm_tokens_stages(tok, ctas) < 3) continue;
                if (c->tune.token_ctas > 0 && ctas != std::min(uint32_t(c->tune.token_ctas), 2u) && gemm_tokens_stages(tok, 2) >= 3) continue;
                int held = int(sms) * int(ctas);
                if (s > 1 && (held = layer_token_capacity(c, kind, tok, s, ctas)) <= 0) continue;
                const double waves = ceil(ctas_all / held);
                const double on_sm = ctas == 1 ? waves : std::max(ceil(ctas_all / sms), ctas_all * 2 > sms ? 2.0 : 1.0);
                double us = 2.5 + std::max(memory, on_sm * per * stage / 130e3) + epilogue * waves + (waves - 1) * 1.5;
                if (wanted) us *= 1e-6;   // the knob's choice wins
                if (us < best.us) best = {false, tok, s, ctas, us};
            }
        }
    }
    return best;
}
// The estimates take a few microseconds; a program repeats the same few sizes.
ProductPlan layer_plan(mmeb200_ctx* c, uint32_t kind, uint32_t M, uint32_t N, uint32_t kb, uint32_t out_bytes, bool rows_aligned) {
    const uint64_t key[2] = {uint64_t(M) << 32 | N, uint64_t(kb) << 32 | kind << 8 | out_bytes << 4 | uint32_t(rows_aligned) << 1 | 1u};
    auto& slot = c->plans[(key[0] * 0x9E3779B97F4A7C15ull ^ key[1] * 0xC2B2AE3D27D4EB4Full) >> 58];
    if (slot.key[0] != key[0] || slot.key[1] != key[1]) {
        slot.plan = layer_make_plan(c, kind, M, N, kb, out_bytes, rows_aligned);
        slot.key[0] = key[0];
        slot.key[1] = key[1];
    }
    return slot.plan;
}

// Few tokens or few tiles: the cluster kernel (gemm_tokens.cuh).
int layer_token_product(mmeb200_ctx* c, uint32_t kind, const TmaOperand& ox, const TmaOperand& ow, const LayerPads& pads, const ProductPlan& plan, TokenGemmParams& p) {
    p.num_k_blocks = uint32_t((ox.inner + kRowBytes - 1) / kRowBytes);
    p.tok = plan.tok;
    p.splits = plan.splits;
    p.ctas = plan.ctas;
    p.idesc = kind == KIND_I8 ? make_instr_desc_i8(kBlockM, p.tok) : make_instr_desc(ow.hw_fmt, ox.hw_fmt, 0, 0, kBlockM, p.tok);
    p.status = c->d_status;
    TRY(encode_tiled(c, &p.tm_w, ow, kRowBytes, kBlockM));
    TRY(encode_tiled(c, &p.tm_x, ox, kRowBytes, p.tok));
    TRY(pads.launch(c));
    for (; uint64_t(p.m_tile0) * p.tok < p.M; p.m_tile0 += kTokenTilesY) TRY(launch_status(c, launch_gemm_tokens(launch_env(c), kind, p)));
    return 0;
}

// Whether a tensor map can describe the output.
bool layer_tma_output(const TokenGemmParams& t, const mmeb200_ctx* c, TmaOperand* out = nullptr) {
    TmaOperand od;
    od.ptr = t.out; od.elem = t.out_bf16 ? 2 : 4; od.inner = t.N; od.rows = t.M; od.row_stride = t.out_ld;
    if (out) *out = od;
    return c->tune.tma_store != 0 && (uint64_t(t.N) * od.elem) % 16 == 0 && tma_compatible(od);
}

// Many tiles: the CTA-pair kernel of the other GEMMs, with the scaling epilogue.
int layer_pair_product(mmeb200_ctx* c, uint32_t kind, const TmaOperand& ox, const TmaOperand& ow, const LayerPads& pads, const TokenGemmParams& t) {
    GemmParams p;
    memset(&p, 0, sizeof p);
    p.M = t.M; p.N = t.N; p.K = uint32_t(ox.inner);
    p.elem_bytes = 1; p.block_k = kRowBytes; p.num_k_blocks = uint32_t((ox.inner + kRowBytes - 1) / kRowBytes);
    p.m_tiles = (p.M + 255) / 256; p.n_tiles = (p.N + 255) / 256; p.batches = 1; p.split_k = 1; p.tile_n = 256;
    p.raster_gm = plan_raster_group(256, p.K, 1);
    if (c->tune.raster_gm > 0) p.raster_gm = uint32_t(c->tune.raster_gm);
    for (int i = 0; i < 3; ++i) { p.bsz[i] = 1; p.a_bcast[i] = 1; p.b_bcast[i] = 1; }
    p.a_mode = A_TILED;
    p.idesc = kind == KIND_I8 ? make_instr_desc_i8(256, 256) : make_instr_desc(ox.hw_fmt, ow.hw_fmt, 0, 0, 256, 256);
    p.out = t.out; p.out_dtype = t.out_bf16 ? DT_BF16 : DT_FP32; p.out_ld = t.out_ld;
    p.scale = t.scale; p.scaled = t.scaled; p.status = c->d_status;
    TRY(encode_tiled(c, &p.tm_a, ox, kRowBytes, kBlockM));
    TRY(encode_tiled(c, &p.tm_b, ow, kRowBytes, 128));
    p.b_cta_bytes = 128 * kRowBytes;
    TmaOperand od;
    if (layer_tma_output(t, c, &od) && encode_tiled(c, &p.tm_out, od, kRowBytes / od.elem, 32, od.elem == 2 ? 2 : 0) == 0) p.tma_store = 1;
    bool two_groups = p.num_k_blocks <= 12;
    if (c->tune.epi_groups > 0) two_groups = c->tune.epi_groups == 2;
    TRY(pads.launch(c));
    return launch_status(c, launch_gemm_pair_scaled(launch_env(c), kind, two_groups ? 2 : 1, p, uint64_t(p.m_tiles) * p.n_tiles));
}

int run_scaled_gemm(mmeb200_ctx* c, mmeb200_tensor* out, const mmeb200_tensor* x, const mmeb200_tensor* x_scale, const mmeb200_tensor* w,
                    const mmeb200_tensor* w_scale, const mmeb200_tensor* bias, int op) {
    TRY(layer_check(c, out, "output", true, false));
    TRY(layer_check(c, x, "x", false, true));
    TRY(layer_check(c, w, "w", false, true));
    if (op != MMEB200_OP_ABT) return c->fail(MMEB200_ERR_UNSUPPORTED, "operation %d: scaled products take both operands with the common dimension contiguous (ABT)", op);
    for (int d = 2; d < 5; ++d)
        if (out->sizes[d] != 1 || x->sizes[d] != 1 || w->sizes[d] != 1) return c->fail(MMEB200_ERR_UNSUPPORTED, "scaled products are 2-D");
    const bool i8 = x->dtype == MMEB200_INT8;
    if (i8 != (w->dtype == MMEB200_INT8)) return c->fail(MMEB200_ERR_UNSUPPORTED, "int8 and fp8 operands cannot be mixed");
    if (!i8) {
        for (const mmeb200_tensor* t : {x, w})
            if (!((t->dtype == DT_FP8_143 && t->inf_nan_mode == MMEB200_INFNAN_MINIMAL) || (t->dtype == DT_FP8_152 && t->inf_nan_mode == MMEB200_INFNAN_FULL)))
                return c->fail(MMEB200_ERR_UNSUPPORTED, "scaled products take fp8 operands whose Inf/NaN convention the tensor cores share (1-4-3 'minimal', 1-5-2 'full')");
        if (x->fp_bias > 30 || w->fp_bias > 30) return c->fail(MMEB200_ERR_INVALID_ARG, "exponent biases %u, %u are out of range", x->fp_bias, w->fp_bias);
        if (c->acc_mode == MMEB200_ACC_CHIP_EXACT) return c->fail(MMEB200_ERR_UNSUPPORTED, "scaled fp8 products accumulate on the tensor cores only");
    }
    const uint64_t K = x->sizes[0], M = x->sizes[1], N = w->sizes[1];
    if (w->sizes[0] != K) return c->fail(MMEB200_ERR_INVALID_ARG, "Common dim doesnt match between input A\\B");
    if (out->sizes[0] != N || out->sizes[1] != M) return c->fail(MMEB200_ERR_INVALID_ARG, "output width doesnt match to inputB width");
    // 131071 products of -128 * -128 are the most an int32 accumulator holds
    if (i8 && K > 131071) return c->fail(MMEB200_ERR_UNSUPPORTED, "int8 products have at most 131071 terms, got %llu", (unsigned long long) K);
    TRY(layer_check_scale(c, x_scale, "x_scale", M, true));
    TRY(layer_check_scale(c, w_scale, "w_scale", N, true));
    if (bias) {
        TRY(layer_check(c, bias, "bias", true, false));
        TRY(layer_check_vector(c, bias, "bias", N));
    }
    TRY(layer_check_distinct(c, out, "output"));
    for (const mmeb200_tensor* t : {x, w, x_scale, w_scale, bias}) TRY(layer_check_overlap(c, out, "output", t, "an input", false));
    if (M == 0 || N == 0) return 0;
    LayerStage st(c);
    const mmeb200_tensor *tx = x, *tw = w, *txs = x_scale, *tws = w_scale, *tb = bias, *to = out;
    TRY(st.begin({x, w, x_scale, w_scale, bias, out}));
    if (K) {
        TRY(st.add(&tx, true, false));
        TRY(st.add(&tw, true, false));
    }
    TRY(st.add(&txs, true, false));
    TRY(st.add(&tws, true, false));
    TRY(st.add(&tb, true, false));
    TRY(st.add(&to, false, true));
    TokenGemmParams p;
    memset(&p, 0, sizeof p);
    p.M = uint32_t(M); p.N = uint32_t(N);
    p.scale = i8 ? 1.0f : ldexpf(1.0f, ((x->dtype == DT_FP8_143 ? 7 : 15) - int(x->fp_bias)) + ((w->dtype == DT_FP8_143 ? 7 : 15) - int(w->fp_bias)));
    p.scaled.row_scale = static_cast<const float*>(txs->data);
    p.scaled.col_scale = static_cast<const float*>(tws->data);
    p.scaled.row_stride = num_elems(x_scale) == 1 ? 0 : 1;
    p.scaled.col_stride = num_elems(w_scale) == 1 ? 0 : 1;
    p.scaled.col_bias = tb ? tb->data : nullptr;
    p.scaled.bias_bf16 = tb && tb->dtype == DT_BF16;
    p.out = to->data; p.out_bf16 = to->dtype == DT_BF16; p.out_ld = to->strides[1];
    if (K == 0) {
        TRY(launch_status(c, launch_gemm_empty_sum(launch_env(c), p)));
        return st.finish();
    }
    const uint32_t kind = i8 ? KIND_I8 : KIND_F8;
    TmaOperand ox, ow;
    const bool x_fits = layer_operand(tx, &ox), w_fits = layer_operand(tw, &ow);
    const ProductPlan plan = layer_plan(c, kind, p.M, p.N, uint32_t((K + kRowBytes - 1) / kRowBytes), p.out_bf16 ? 2 : 4, layer_tma_output(p, c));
    LayerScratchUse use(LayerScratchMark{c});
    LayerPads pads;
    if (!x_fits || !w_fits) {
        const size_t xb = x_fits ? 0 : LayerPads::bytes(ox), wb = w_fits ? 0 : LayerPads::bytes(ow);
        void* scratch = nullptr;
        TRY(layer_scratch(c, xb + wb, "operands need 16-byte aligned rows", &scratch));
        use.begin();
        if (!x_fits) pads.add(&ox, static_cast<uint8_t*>(scratch));
        if (!w_fits) pads.add(&ow, static_cast<uint8_t*>(scratch) + xb);
    }
    TRY(plan.pair ? layer_pair_product(c, kind, ox, ow, pads, p) : layer_token_product(c, kind, ox, ow, pads, plan, p));
    TRY(use.end());
    return st.finish();
}

// No C++ exception leaves the library.
template <typename F>
int layer_entry(mmeb200_ctx* c, F&& body) {
    if (!c) return MMEB200_ERR_INVALID_ARG;
    try {
        DeviceGuard guard(c->device);
        return body();
    } catch (...) {
        return MMEB200_ERR_CUDA;
    }
}

}  // namespace

extern "C" int mmeb200_rms_norm(mmeb200_ctx* c, mmeb200_tensor* out, mmeb200_tensor* scale, mmeb200_tensor* sum, const mmeb200_tensor* x,
                                const mmeb200_tensor* residual, const mmeb200_tensor* gamma, float eps, int scale_mode) {
    return layer_entry(c, [&] { return run_rms_norm(c, out, scale, sum, x, residual, gamma, eps, scale_mode, true); });
}
extern "C" int mmeb200_rms_norm_grad(mmeb200_ctx* c, mmeb200_tensor* dx, mmeb200_tensor* dgamma, const mmeb200_tensor* dy, const mmeb200_tensor* x,
                                     const mmeb200_tensor* gamma, const mmeb200_tensor* dsum, float eps, mmeb200_tensor* workspace) {
    return layer_entry(c, [&] { return run_rms_norm_grad(c, dx, dgamma, dy, x, gamma, dsum, eps, workspace); });
}
extern "C" size_t mmeb200_rms_norm_grad_workspace(const mmeb200_ctx* c, uint64_t rows, uint64_t cols) {
    if (!c || rows >= (uint64_t(1) << 31) || cols >= (uint64_t(1) << 31)) return 0;
    DeviceGuard guard(c->device);
    return size_t(norm_grad_blocks(c->device, c->sm_count, uint32_t(rows), uint32_t(cols))) * cols * sizeof(float);
}
extern "C" int mmeb200_quantize(mmeb200_ctx* c, mmeb200_tensor* out, mmeb200_tensor* scale, const mmeb200_tensor* x, int op, int scale_mode) {
    return layer_entry(c, [&] { return run_quantize(c, out, scale, x, op, scale_mode); });
}
extern "C" int mmeb200_scaled_gemm(mmeb200_ctx* c, mmeb200_tensor* out, const mmeb200_tensor* x, const mmeb200_tensor* x_scale, const mmeb200_tensor* w,
                                   const mmeb200_tensor* w_scale, const mmeb200_tensor* bias, int op) {
    return layer_entry(c, [&] { return run_scaled_gemm(c, out, x, x_scale, w, w_scale, bias, op); });
}
