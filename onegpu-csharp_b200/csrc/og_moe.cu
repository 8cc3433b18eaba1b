// A whole mixture-of-experts layer for a few tokens on int8 weights, with its argument checks and C ABI.
//
//   logits[t][e] = sum_d x[t][d] router[e][d],  p = softmax over the experts
//   the top_k experts of a token by p (ties to the lowest index), w = p, or p / (sum of the chosen p) when normalized
//   u = scale_in[e][j] sum_d w_in[e][j][d] x[t][d];   h[j] = activation(u[j]) u[F + j]  (gated), activation(u[j])
//   y[t][d] = residual[t][d] + sum over the chosen e of w_e scale_out[e][d] sum_j w_out[e][d][j] h[j]
//
// How the sums are held: og_moe_fused.cu. A NaN logit ranks below every number.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <vector>

#include "og_gemm.h"
#include "og_host.h"
#include "og_moe.h"
#include "og_ptx.cuh"

// ---- host layer ------------------------------------------------------------------------------------------------------

using namespace og_host;

struct og_int8_moe {
    og_device* device = nullptr;
    std::string last = "none";
    std::vector<void*> buffers;  // workspaces, the latest last; older ones live until destroy (recorded work names them)
    int64_t bytes = 0;
    og::MoeCounts* counts = nullptr;  // of the fused kernel
    int late_barrier = 0;             // watchdog self-test of the next layer recorded, 0 for none
    uint64_t limit_ns = 0;
};

namespace {

const char* kMoe = "Int8Moe";

void require_float(const og_buffer* b, const char* arg) {
    if (b->type != OG_F32 && b->type != OG_F16)
        shape(kMoe, arg, std::string("element type ") + type_name(b->type) + " is not supported; use Single or Half");
}

void require(const og_buffer* b, const char* arg, int32_t type) {
    if (b->type != type)
        shape(kMoe, arg, std::string("element type ") + type_name(b->type) + " is not supported; use " + type_name(type));
}

void between(const char* arg, int32_t v, int32_t low, int32_t high) {
    if (v < low || v > high)
        shape(kMoe, arg, std::to_string(v) + " is outside " + std::to_string(low) + ".." + std::to_string(high));
}

void need(const og_buffer* b, const char* arg) {
    if (b == nullptr || b->ptr == nullptr) null_arg(kMoe, arg);
}

template <class T>
T* at(const og_buffer* b, int32_t offset) {
    return reinterpret_cast<T*>(static_cast<uint8_t*>(b->ptr) + static_cast<int64_t>(offset) * elem_size(b->type));
}

// The checks; false when there is nothing to do (no tokens).
bool check_moe(const og_moe_problem* p, const og_buffer* x, const og_buffer* router, const og_buffer* w_in,
               const og_buffer* w_in_scale, const og_buffer* w_out, const og_buffer* w_out_scale, const og_buffer* y,
               const og_buffer* residual, const og_buffer* ids, const og_buffer* weights) {
    need(x, "x");
    need(router, "router");
    need(w_in, "wIn");
    need(w_in_scale, "wInScale");
    need(w_out, "wOut");
    need(w_out_scale, "wOutScale");
    need(y, "y");
    if (p == nullptr) null_arg(kMoe, "problem");
    require_float(x, "x");
    require_float(router, "router");
    require(w_in, "wIn", OG_S8);
    require(w_in_scale, "wInScale", OG_F32);
    require(w_out, "wOut", OG_S8);
    require(w_out_scale, "wOutScale", OG_F32);
    require(y, "y", x->type);
    between("Tokens", p->tokens, 0, og::MOE_MAX_TOKENS);
    between("ModelSize", p->model_size, 1, og::MOE_MAX_SIZE);
    between("ExpertSize", p->expert_size, 1, og::MOE_MAX_SIZE);
    between("Experts", p->experts, 1, og::MOE_MAX_EXPERTS);
    between("TopK", p->top_k, 1, std::min(p->experts, og::MOE_MAX_TOP_K));
    between("Activation", p->activation, OG_ACTIVATION_NONE, OG_ACTIVATION_SILU);
    const int64_t t = p->tokens, d = p->model_size, e = p->experts;
    const int64_t up = static_cast<int64_t>(p->gated ? 2 : 1) * p->expert_size, f = p->expert_size;
    range(kMoe, "x", x->length, p->offset_x, t * d);
    range(kMoe, "router", router->length, p->offset_router, e * d);
    range(kMoe, "wIn", w_in->length, p->offset_in, e * up * d);
    range(kMoe, "wInScale", w_in_scale->length, p->offset_in_scale, e * up);
    range(kMoe, "wOut", w_out->length, p->offset_out, e * d * f);
    range(kMoe, "wOutScale", w_out_scale->length, p->offset_out_scale, e * d);
    range(kMoe, "y", y->length, p->offset_y, t * d);
    if (residual != nullptr) {
        need(residual, "residual");
        require(residual, "residual", y->type);
        range(kMoe, "residual", residual->length, p->offset_residual, t * d);
        const uint8_t* r0 = at<uint8_t>(residual, p->offset_residual);
        const uint8_t* y0 = at<uint8_t>(y, p->offset_y);
        const int64_t bytes = t * d * elem_size(y->type);
        if (r0 != y0 && r0 < y0 + bytes && y0 < r0 + bytes)
            shape(kMoe, "residual", "overlaps y without being the same elements");
    }
    if (ids != nullptr) {
        need(ids, "expertIds");
        require(ids, "expertIds", OG_I32);
        range(kMoe, "expertIds", ids->length, p->offset_ids, t * p->top_k);
    }
    if (weights != nullptr) {
        need(weights, "expertWeights");
        require(weights, "expertWeights", OG_F32);
        range(kMoe, "expertWeights", weights->length, p->offset_weights, t * p->top_k);
    }
    return p->tokens > 0;
}

int64_t round256(int64_t v) { return (v + 255) & ~int64_t(255); }

// Carves the layer's workspace out of the instance's, growing it geometrically.
void bind_workspace(og_int8_moe* m, og::MoeLaunch& L) {
    const int64_t pairs = static_cast<int64_t>(L.tokens) * L.top_k;
    const og::MoeFusedSizes s = og::moe_fused_sizes(L);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round256(bytes);
        return here;
    };
    const int64_t ids = take(pairs * 4), weights = take(pairs * 4), hidden = take(s.hidden);
    const int64_t logits = take(s.logits), x = take(s.x_digits), h = take(s.h_digits), outputs = take(s.outputs);
    const int64_t x_most = take(s.x_most), h_most = take(s.h_most), segments = take(s.segments);
    if (m->bytes < at) {
        const int64_t len = std::max(at, std::max<int64_t>(int64_t(1) << 20, 2 * m->bytes));
        void* p = nullptr;
        check_cuda(cudaMalloc(&p, static_cast<size_t>(len)), "Int8Moe workspace");
        m->buffers.push_back(p);
        m->bytes = len;
    }
    uint8_t* base = static_cast<uint8_t*>(m->buffers.back());
    L.ids = reinterpret_cast<int32_t*>(base + ids);
    L.weights = reinterpret_cast<float*>(base + weights);
    L.hidden = reinterpret_cast<float*>(base + hidden);
    L.logits = reinterpret_cast<double*>(base + logits);
    L.x_digits = base + x;
    L.h_digits = base + h;
    L.x_most = reinterpret_cast<uint32_t*>(base + x_most);
    L.h_most = reinterpret_cast<uint32_t*>(base + h_most);
    L.outputs = reinterpret_cast<float*>(base + outputs);
    L.segments = reinterpret_cast<long long*>(base + segments);
}

}  // namespace

extern "C" {

OG_API og_status og_int8_moe_create(og_device* d, og_int8_moe** out) {
    return guard([&] {
        if (d == nullptr) null_arg(kMoe, "device");
        if (out == nullptr) null_arg(kMoe, "out");
        use(d);
        void* p = device_zeros(sizeof(og::MoeCounts), "Int8Moe counts");
        auto* m = new og_int8_moe();
        m->device = d;
        m->counts = static_cast<og::MoeCounts*>(p);
        *out = m;
    });
}

OG_API og_status og_int8_moe_destroy(og_int8_moe* m) {
    return guard([&] {
        if (m == nullptr) return;
        use(m->device);
        cudaStreamSynchronize(m->device->stream);
        for (void* p : m->buffers) cudaFree(p);
        cudaFree(m->counts);
        delete m;
    });
}

OG_API og_status og_int8_moe_last_kernel(og_int8_moe* m, char* buffer, uint64_t capacity) {
    return guard([&] {
        if (m == nullptr) throw OgError{OG_ERROR_INVALID_HANDLE, kMoe, "moe", "null handle", "", "", ""};
        if (buffer == nullptr || capacity == 0) return;
        const size_t n = std::min(static_cast<size_t>(capacity) - 1, m->last.size());
        m->last.copy(buffer, n);
        buffer[n] = 0;
    });
}

OG_API og_status og_int8_moe_watchdog_selftest(og_int8_moe* m, int32_t barrier, uint32_t limit_us) {
    return guard([&] {
        if (m == nullptr) throw OgError{OG_ERROR_INVALID_HANDLE, kMoe, "moe", "null handle", "", "", ""};
        if (barrier < 1 || barrier > 4)
            throw OgError{OG_ERROR_ARGUMENT_RANGE, kMoe, "barrier", "the layer's barriers are 1 .. 4", "", "", ""};
        if (limit_us < 1 || limit_us > 500000)
            throw OgError{OG_ERROR_ARGUMENT_RANGE, kMoe, "limitMicroseconds",
                          "the self-test wait limit is 1 .. 500000 microseconds", "", "", ""};
        m->late_barrier = barrier;
        m->limit_ns = uint64_t(limit_us) * 1000;
    });
}

OG_API og_status og_int8_moe_check(const og_moe_problem* p, const og_buffer* x, const og_buffer* router,
                                   const og_buffer* w_in, const og_buffer* w_in_scale, const og_buffer* w_out,
                                   const og_buffer* w_out_scale, const og_buffer* y, const og_buffer* residual,
                                   const og_buffer* ids, const og_buffer* weights) {
    return guard([&] { check_moe(p, x, router, w_in, w_in_scale, w_out, w_out_scale, y, residual, ids, weights); });
}

OG_API og_status og_int8_moe_encode(og_int8_moe* m, og_encoder* enc, const og_moe_problem* p, const og_buffer* x,
                                    const og_buffer* router, const og_buffer* w_in, const og_buffer* w_in_scale,
                                    const og_buffer* w_out, const og_buffer* w_out_scale, const og_buffer* y,
                                    const og_buffer* residual, const og_buffer* ids, const og_buffer* weights) {
    return guard([&] {
        if (m == nullptr) throw OgError{OG_ERROR_INVALID_HANDLE, kMoe, "moe", "null handle", "", "", ""};
        if (enc == nullptr) null_arg(kMoe, "encoder");
        if (enc->device != m->device)
            throw OgError{OG_ERROR_INVALID_HANDLE, kMoe, "encoder", "the encoder belongs to another device", "", "", ""};
        if (!check_moe(p, x, router, w_in, w_in_scale, w_out, w_out_scale, y, residual, ids, weights)) {
            m->last = "none";
            return;
        }
        use(m->device);
        og::MoeLaunch L = {};
        L.tokens = p->tokens;
        L.model = p->model_size;
        L.expert = p->expert_size;
        L.experts = p->experts;
        L.top_k = p->top_k;
        L.activation = p->activation;
        L.gated = p->gated != 0;
        L.normalize = p->normalize != 0;
        L.x_half = x->type == OG_F16;
        L.router_half = router->type == OG_F16;
        L.x = at<void>(x, p->offset_x);
        L.router = at<void>(router, p->offset_router);
        L.w_in = at<int8_t>(w_in, p->offset_in);
        L.in_scale = at<float>(w_in_scale, p->offset_in_scale);
        L.w_out = at<int8_t>(w_out, p->offset_out);
        L.out_scale = at<float>(w_out_scale, p->offset_out_scale);
        L.y = at<void>(y, p->offset_y);
        L.residual = residual != nullptr ? at<void>(residual, p->offset_residual) : nullptr;
        L.ids_out = ids != nullptr ? at<int32_t>(ids, p->offset_ids) : nullptr;
        L.weights_out = weights != nullptr ? at<float>(weights, p->offset_weights) : nullptr;
        L.counts = m->counts;
        L.error_flag = m->device->status;
        L.num_sms = m->device->sm_count;
        L.wait_limit_ns = m->late_barrier != 0 ? m->limit_ns : og::OG_WAIT_LIMIT_NS;
        L.late_barrier = m->late_barrier;
        L.late_ns = 3 * L.wait_limit_ns;
        bind_workspace(m, L);
        cudaError_t err;
        auto fn = og::prepare_moe_fused(L, &err);  // tensor maps built now, at record time
        check_cuda(err, "Int8Moe tensor maps");
        m->last = og::moe_aligned(L) ? "fused" : "fused-unaligned";
        enc->ops.push_back(std::move(fn));
        m->late_barrier = 0;
        enc->dispatches += 1;
    });
}

}  // extern "C"
