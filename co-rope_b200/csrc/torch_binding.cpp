// Host path of the Python entry points: argument checks, layouts, workspaces and autograd nodes in C++, calling the C ABI of
// include/corope_b200.h.  A forward + backward through Python (ctypes calls, torch.autograd.Function) cost 210 us of host time per
// step, more than the kernels of every small shape take; this path costs a fraction of it.
//
// The checks and their exceptions are those of the reference's entry points: fused-rope/fused_rope_attn.py:657-661,
// fused-rope/flash_attn_v2_triton.py:517-521, corope-exp/flash_attn_co_rope_gqa_triton.py:407-425.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <mutex>
#include <stdexcept>

#include "../../include/corope_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct AssertError : std::runtime_error {   // surfaces as AssertionError
    using std::runtime_error::runtime_error;
};
struct ValueError : std::runtime_error {    // surfaces as ValueError
    using std::runtime_error::runtime_error;
};
void require(bool ok, const char* what) {
    if (!ok) throw AssertError(what);
}
void require_value(bool ok, const std::string& what) {
    if (!ok) throw ValueError(what);
}

// ------------------------------------------------------------------------------------------------ device status
// The status word of one GPU and its pinned host mirror.  The kernels write the mirror themselves when they fail, so looking at
// it before a call costs one host load and no copy is enqueued behind the call.
struct DeviceStatus {
    Tensor word, mirror;
    int* word_ptr = nullptr;
    volatile int* mirror_ptr = nullptr;
};
constexpr int kMaxDevices = 64;
DeviceStatus g_status[kMaxDevices];
std::once_flag g_status_once[kMaxDevices];

DeviceStatus& device_status(int index) {
    TORCH_CHECK(index >= 0 && index < kMaxDevices, "corope_b200: device index out of range");
    std::call_once(g_status_once[index], [index] {
        DeviceStatus& st = g_status[index];
        st.word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, index));
        st.mirror = at::zeros({1}, at::TensorOptions().dtype(at::kInt)).pin_memory();
        st.word_ptr = st.word.data_ptr<int>();
        st.mirror_ptr = st.mirror.data_ptr<int>();
        const int rc = corope_status_mirror_register(st.word_ptr, const_cast<int*>(st.mirror_ptr));
        TORCH_CHECK(rc == 0, "corope_b200: the status mirror could not be registered (", rc, ")");
    });
    return g_status[index];
}

std::string status_message(int v) {   // as _ext._status_message
    std::string text;
    auto add = [&](int bit, const char* what) {
        if (v & bit) text += (text.empty() ? "" : "; ") + std::string(what);
    };
    add(COROPE_DEV_WAIT_EXPIRED, "a bounded device-side wait expired (results of that call and of later calls are undefined)");
    add(COROPE_DEV_RANGE, "a gradient term left the value range of the 16-bit Co-RoPE backward and was clamped (results of that call are inaccurate)");
    add(COROPE_DEV_BAD_INDEX, "a block table entry, length or position of a cache operator pointed outside its tensor (it was not followed; the tokens concerned were left out)");
    return text;
}

// Raises if an earlier call on this device left the status word set; clears it first.
void look_at_status(DeviceStatus& st, cudaStream_t stream) {
    const int v = *st.mirror_ptr;
    if (v == 0) return;
    corope_status_mirror_clear(st.word_ptr, const_cast<int*>(st.mirror_ptr), stream);
    char text[64];
    snprintf(text, sizeof text, "corope_b200: an earlier kernel reported device status 0x%x: ", v);
    throw std::runtime_error(text + status_message(v));
}

void raise_for_status(int rc, const char* what) {
    if (rc == 0) return;
    const std::string msg = corope_status_string(rc);
    if (rc == COROPE_ERR_BAD_HEAD_DIM) throw AssertError(std::string(what) + ": " + msg);
    if (rc == COROPE_ERR_BAD_GROUP) throw ValueError(std::string(what) + ": " + msg);
    throw std::runtime_error(std::string(what) + " failed with status " + std::to_string(rc) + ": " + msg);
}

// ------------------------------------------------------------------------------------------------ tensors
int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return COROPE_DTYPE_F32;
        case at::kBFloat16: return COROPE_DTYPE_BF16;
        case at::kHalf: return COROPE_DTYPE_F16;
        default: return -1;
    }
}
void require_cuda(const Tensor& t) {
    if (!t.is_cuda())
        throw std::runtime_error("corope_b200 runs on CUDA tensors only (got a " + c10::DeviceTypeName(t.device().type(), true) +
                                 " tensor); there is no CPU path.");
}
// `t` itself when the kernels can take its layout (unit stride along the head dimension, no overlapping or broadcast strides),
// else a contiguous copy.
Tensor kernel_layout(const Tensor& t) {
    const auto st = t.strides();
    if (st[3] == 1 && st[0] > 0 && st[1] > 0 && st[2] >= t.size(3)) return t;
    return t.contiguous();
}
// Outputs and gradients: laid out like the input, or contiguous (the entry point that takes theta)
Tensor new_like(const Tensor& t, bool contiguous) { return contiguous ? at::empty(t.sizes(), t.options()) : at::empty_like(t); }
void set_strides(int64_t (&dst)[3], const Tensor& t) {
    const auto st = t.strides();
    dst[0] = st[0]; dst[1] = st[1]; dst[2] = st[2];
}

// Everything one library call needs besides its tensors.
struct Call {
    c10::cuda::CUDAGuard guard;
    cudaStream_t stream;
    DeviceStatus& status;
    explicit Call(const Tensor& t) : guard(t.device()), stream(at::cuda::getCurrentCUDAStream(t.device().index())), status(device_status(t.device().index())) {
        look_at_status(status, stream);
    }
};
struct Workspace {
    Tensor buf;
    size_t bytes;
    Workspace(int op, int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D, int dtype, const Tensor& like) {
        bytes = corope_workspace_bytes_any_n(op, (int)B, (int)Hq, (int)Hkv, (int)N, (int)D, dtype);
        auto allocate = [&] { buf = at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(at::kByte)); };
        try {
            allocate();
        } catch (const c10::OutOfMemoryError&) {   // the split copies are for speed: without them a call runs on the CUDA cores
            const size_t least = corope_workspace_bytes(op, (int)B, (int)Hq, (int)Hkv, (int)N, (int)D, dtype);
            if (least >= bytes) throw;
            bytes = least;
            allocate();
        }
    }
    void* ptr() const { return buf.data_ptr(); }
};
Tensor new_rows(const Tensor& like, int64_t B, int64_t H, int64_t N) { return at::empty({B, H, N}, like.options().dtype(at::kFloat)); }

// RoPE tables: fp32, unit column stride, one row stride for both
struct Tables {
    Tensor cos, sin;
    int64_t stride;
};
Tables tables(const Tensor& freqs_cos, const Tensor& freqs_sin, int64_t N, int64_t D) {
    require_value(freqs_cos.dim() == 2 && freqs_cos.sizes() == freqs_sin.sizes(), "freqs_cos and freqs_sin must be 2-D tensors of the same shape");
    if (freqs_cos.size(0) < N || freqs_cos.size(1) < D / 2) {
        std::ostringstream os;
        os << "RoPE tables must cover [N, D/2] = [" << N << ", " << D / 2 << "], got (" << freqs_cos.size(0) << ", " << freqs_cos.size(1) << ")";
        throw ValueError(os.str());
    }
    auto fix = [](const Tensor& t) {
        require_cuda(t);
        return t.scalar_type() == at::kFloat && t.stride(1) == 1 ? t : t.to(at::kFloat).contiguous();
    };
    Tables r{fix(freqs_cos), fix(freqs_sin), 0};
    if (r.cos.stride(0) != r.sin.stride(0)) r.cos = r.cos.contiguous(), r.sin = r.sin.contiguous();
    r.stride = r.cos.stride(0);
    return r;
}

// checks shared by the fused-RoPE and the plain entry points
void check_mha(const Tensor& q, const Tensor& k, const Tensor& v, bool grouped) {
    require(q.dim() >= 1 && k.dim() >= 1 && v.dim() >= 1, "q, k, v must be 4-D tensors");
    const int64_t D = k.size(-1);
    require(q.size(-1) == D && D == v.size(-1), "q, k and v must share one head dimension");
    require(D == 32 || D == 64 || D == 128, "corope_b200 supports head dims (32, 64, 128)");
    require(q.dim() == 4 && k.sizes() == v.sizes(), "q, k, v must be [B, H, N, D] tensors, k and v of one shape");
    if (grouped) {
        require(k.dim() == 4 && q.size(0) == k.size(0) && q.size(2) == k.size(2), "q and k must agree in batch and sequence length");
    } else {
        require(q.sizes() == k.sizes(), "q, k and v must share one shape");
    }
    require(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && dtype_code(q) >= 0,
            "q, k, v must share one dtype out of float32, bfloat16, float16");
    if (grouped) require(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "number of query heads must be a multiple of the number of K / V heads");
    for (const Tensor* t : {&q, &k, &v}) require_cuda(*t);
}

// ------------------------------------------------------------------------------------------------ attention with rotation or without
enum Kind { kRope, kTheta, kFlash };

struct Saved {
    Tensor q, k, v, o, m;
    Tables tab;   // kRope only
};

Saved mha_forward(Kind kind, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, bool causal, double sm_scale, const Tensor& freqs_cos,
                  const Tensor& freqs_sin, double theta) {
    check_mha(q_in, k_in, v_in, kind == kFlash);
    const int64_t B = q_in.size(0), Hq = q_in.size(1), N = q_in.size(2), D = q_in.size(3), Hkv = k_in.size(1);
    const int dt = dtype_code(q_in);
    Saved s;
    if (kind == kRope) s.tab = tables(freqs_cos, freqs_sin, N, D);
    Call call(q_in);
    s.q = kernel_layout(q_in);
    s.k = kernel_layout(k_in);
    s.v = kernel_layout(v_in);
    s.o = new_like(s.q, kind == kTheta);
    s.m = new_rows(s.q, B, Hq, N);
    const int op = kind == kRope ? COROPE_OP_ROPE_FWD : kind == kTheta ? COROPE_OP_ROPE_FWD_FREQS : COROPE_OP_FLASH_FWD;
    Workspace ws(op, B, Hq, Hkv, N, D, dt, s.q);
    corope_strides_t st{};
    set_strides(st.q, s.q);
    set_strides(st.k, s.k);
    set_strides(st.v, s.v);
    set_strides(st.o, s.o);
    float* m = s.m.data_ptr<float>();
    const int Bi = (int)B, Hi = (int)Hq, Ni = (int)N, Di = (int)D, ca = causal ? 1 : 0;
    const float sc = (float)sm_scale;
    if (kind == kRope) {
        raise_for_status(corope_rope_attn_fwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.tab.cos.data_ptr<float>(),
                                                      s.tab.sin.data_ptr<float>(), s.tab.stride, s.o.data_ptr(), m, Bi, Hi, Ni, Di, dt, ca, sc, ws.ptr(),
                                                      ws.bytes, call.status.word_ptr, call.stream, &st),
                         "corope_rope_attn_fwd");
    } else if (kind == kTheta) {
        raise_for_status(corope_rope_attn_fwd_theta(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), (float)theta, s.o.data_ptr(), m, Bi, Hi, Ni, Di, dt, ca,
                                                    sc, ws.ptr(), ws.bytes, call.status.word_ptr, call.stream, &st),
                         "corope_rope_attn_fwd_theta");
    } else {
        raise_for_status(corope_flash_attn_fwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), m, Bi, Hi, (int)Hkv, Ni, Di, dt, ca,
                                                       sc, ws.ptr(), ws.bytes, call.status.word_ptr, call.stream, &st),
                         "corope_flash_attn_fwd");
    }
    return s;
}

struct Grads {
    Tensor dq, dk, dv;
};

// The reference asserts a contiguous dO, equal strides and N % 128 == 0 (fused_rope_attn.py:727-728, 750); these kernels take any N
// and every tensor's own strides.
Grads mha_backward(Kind kind, const Saved& s, const Tensor& d_out, bool causal, double sm_scale, double theta) {
    const int64_t B = s.q.size(0), Hq = s.q.size(1), N = s.q.size(2), D = s.q.size(3), Hkv = s.k.size(1);
    const int dt = dtype_code(s.q);
    Call call(s.q);
    const Tensor d_o = kernel_layout(d_out);
    TORCH_CHECK(d_o.is_cuda() && d_o.scalar_type() == s.q.scalar_type() && d_o.sizes() == s.o.sizes(), "dO must match o");
    Grads g{new_like(s.q, kind == kTheta), new_like(s.k, kind == kTheta), new_like(s.v, kind == kTheta)};
    const int op = kind == kRope ? COROPE_OP_ROPE_BWD : kind == kTheta ? COROPE_OP_ROPE_BWD_FREQS : COROPE_OP_FLASH_BWD;
    Workspace ws(op, B, Hq, Hkv, N, D, dt, s.q);
    corope_strides_t st;
    set_strides(st.q, s.q);
    set_strides(st.k, s.k);
    set_strides(st.v, s.v);
    set_strides(st.o, s.o);
    set_strides(st.d_o, d_o);
    set_strides(st.dq, g.dq);
    set_strides(st.dk, g.dk);
    set_strides(st.dv, g.dv);
    const float* m = s.m.data_ptr<float>();
    const int Bi = (int)B, Hi = (int)Hq, Ni = (int)N, Di = (int)D, ca = causal ? 1 : 0;
    const float sc = (float)sm_scale;
    if (kind == kRope) {
        raise_for_status(corope_rope_attn_bwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), d_o.data_ptr(), m,
                                                      s.tab.cos.data_ptr<float>(), s.tab.sin.data_ptr<float>(), s.tab.stride, g.dq.data_ptr(), g.dk.data_ptr(),
                                                      g.dv.data_ptr(), Bi, Hi, Ni, Di, dt, ca, sc, ws.ptr(), ws.bytes, call.status.word_ptr, call.stream, &st),
                         "corope_rope_attn_bwd");
    } else if (kind == kTheta) {
        raise_for_status(corope_rope_attn_bwd_theta(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), d_o.data_ptr(), m, (float)theta,
                                                    g.dq.data_ptr(), g.dk.data_ptr(), g.dv.data_ptr(), Bi, Hi, Ni, Di, dt, ca, sc, ws.ptr(), ws.bytes,
                                                    call.status.word_ptr, call.stream, &st),
                         "corope_rope_attn_bwd_theta");
    } else {
        raise_for_status(corope_flash_attn_bwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), d_o.data_ptr(), m, g.dq.data_ptr(),
                                                       g.dk.data_ptr(), g.dv.data_ptr(), Bi, Hi, (int)Hkv, Ni, Di, dt, ca, sc, ws.ptr(), ws.bytes,
                                                       call.status.word_ptr, call.stream, &st),
                         "corope_flash_attn_bwd");
    }
    return g;
}

// ------------------------------------------------------------------------------------------------ Co-RoPE
struct GqaSaved {
    Tensor q, k, v, o, lse2, a_diag;
};

GqaSaved gqa_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, bool causal, double sm_scale, double theta) {
    require_value(causal, "CoRoPE fused kernel supports causal=True only.");
    require_value(q_in.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4, "Expected q, k, v to have shape (batch, heads, seqlen, dim).");
    require_value(k_in.sizes() == v_in.sizes(), "k and v must share the same shape in GQA.");
    require_value(q_in.size(0) == k_in.size(0) && q_in.size(2) == k_in.size(2) && q_in.size(3) == k_in.size(3),
                  "k must align with q along batch/sequence/head_dim.");
    const int64_t B = q_in.size(0), Hq = q_in.size(1), N = q_in.size(2), D = q_in.size(3), Hkv = k_in.size(1);
    require_value(Hkv > 0 && Hq % Hkv == 0, "Number of query heads must be divisible by KV heads.");
    require_value(Hq / Hkv <= 8, "CoRoPE backbone currently limits group_size <= 8 (got " + std::to_string(Hq / Hkv) + ").");
    require_value(q_in.scalar_type() == k_in.scalar_type() && q_in.scalar_type() == v_in.scalar_type() && dtype_code(q_in) >= 0,
                  "q, k, v must share one dtype out of float32, bfloat16, float16.");
    for (const Tensor* t : {&q_in, &k_in, &v_in}) require_cuda(*t);
    const int dt = dtype_code(q_in);
    Call call(q_in);
    GqaSaved s;
    s.q = kernel_layout(q_in);
    s.k = kernel_layout(k_in);
    s.v = kernel_layout(v_in);
    s.o = at::empty_like(s.q);
    s.lse2 = new_rows(s.q, B, Hq, N);
    s.a_diag = new_rows(s.q, B, Hkv, N);
    Workspace ws(COROPE_OP_GQA_FWD, B, Hq, Hkv, N, D, dt, s.q);
    corope_strides_t st{};
    set_strides(st.q, s.q);
    set_strides(st.k, s.k);
    set_strides(st.v, s.v);
    set_strides(st.o, s.o);
    raise_for_status(corope_gqa_fwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), s.lse2.data_ptr<float>(),
                                            s.a_diag.data_ptr<float>(), (int)B, (int)Hq, (int)Hkv, (int)N, (int)D, dt, (float)sm_scale, (float)theta, ws.ptr(),
                                            ws.bytes, call.status.word_ptr, call.stream, &st),
                     "corope_gqa_fwd");
    return s;
}

// dk / dv are summed over each group
Grads gqa_backward(const GqaSaved& s, const Tensor& d_out, double sm_scale, double theta) {
    const int64_t B = s.q.size(0), Hq = s.q.size(1), N = s.q.size(2), D = s.q.size(3), Hkv = s.k.size(1);
    const int dt = dtype_code(s.q);
    Call call(s.q);
    const Tensor d_o = kernel_layout(d_out);
    TORCH_CHECK(d_o.is_cuda() && d_o.scalar_type() == s.q.scalar_type() && d_o.sizes() == s.o.sizes(), "dO must match o");
    Grads g{at::empty_like(s.q), at::empty_like(s.k), at::empty_like(s.v)};
    Workspace ws(COROPE_OP_GQA_BWD, B, Hq, Hkv, N, D, dt, s.q);
    corope_strides_t st;
    set_strides(st.q, s.q);
    set_strides(st.k, s.k);
    set_strides(st.v, s.v);
    set_strides(st.o, s.o);
    set_strides(st.d_o, d_o);
    set_strides(st.dq, g.dq);
    set_strides(st.dk, g.dk);
    set_strides(st.dv, g.dv);
    raise_for_status(corope_gqa_bwd_strided(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.o.data_ptr(), d_o.data_ptr(), s.lse2.data_ptr<float>(),
                                            s.a_diag.data_ptr<float>(), g.dq.data_ptr(), g.dk.data_ptr(), g.dv.data_ptr(), (int)B, (int)Hq, (int)Hkv, (int)N,
                                            (int)D, dt, (float)sm_scale, (float)theta, ws.ptr(), ws.bytes, call.status.word_ptr, call.stream, &st),
                     "corope_gqa_bwd");
    return g;
}

// ------------------------------------------------------------------------------------------------ 8-bit paged cache
using Optional = c10::optional<Tensor>;

struct CacheTensors {   // the attributes of a cache object (kv_cache.py)
    Tensor k, v, k_scale, v_scale;
    Optional weight;
};

void require_shape(const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const Tensor& like, const char* name) {
    require_cuda(t);
    if (t.sizes() != shape || t.scalar_type() != type || t.device() != like.device()) {
        std::ostringstream os;
        os << name << " must be a " << type << " tensor of shape " << shape << " on " << like.device() << ", got " << t.scalar_type() << " " << t.sizes() << " on "
           << t.device();
        throw ValueError(os.str());
    }
}
// no gradient flows through the cache, backwards or forwards: a caller who expects one learns it here
void require_no_grad(std::initializer_list<const Tensor*> ts, const CacheTensors& c) {
    const bool grad_mode = at::GradMode::is_enabled();
    auto check = [grad_mode](const Tensor& t) {
        if (t.unsafeGetTensorImpl()->autograd_meta() == nullptr) return;   // neither
        if (grad_mode && t.requires_grad())
            throw std::runtime_error("corope_b200: the cache operators have no backward pass; call them under torch.no_grad()");
        if (t._fw_grad(0).defined()) throw std::runtime_error("corope_b200: the cache operators have no derivatives; a tensor of the call is a forward-mode dual");
    };
    for (const Tensor* t : ts) check(*t);
    for (const Tensor* t : {&c.k, &c.v, &c.k_scale, &c.v_scale}) check(*t);
    if (c.weight.has_value()) check(*c.weight);
}
// Tensors that a call has written to in place: a backward pass that saved one of them has to find out.
void written(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
void whole_cache_written(const CacheTensors& c) {
    written({&c.k, &c.v, &c.k_scale, &c.v_scale});
    if (c.weight.has_value()) written({&*c.weight});
}

corope_kv_cache_t cache_view(const CacheTensors& c, bool written) {
    for (const Tensor* t : {&c.k, &c.v, &c.k_scale, &c.v_scale}) require_cuda(*t);
    require_value(c.k.dim() == 4 && c.k.sizes() == c.v.sizes() && c.k.scalar_type() == c.v.scalar_type() && c.k.device() == c.v.device(),
                  "cache.k and cache.v must be [num_blocks, Hkv, block_size, D] tensors of one shape, type and device");
    require_value(c.k.scalar_type() == at::kFloat8_e4m3fn || c.k.scalar_type() == at::kChar, "cache.k and cache.v must be float8_e4m3fn or int8");
    const int64_t N = c.k.size(0), H = c.k.size(1), bs = c.k.size(2), D = c.k.size(3);
    require(D == 32 || D == 64 || D == 128, "corope_b200 supports head dims (32, 64, 128)");
    require_value(bs >= 16 && bs <= 256 && (bs & (bs - 1)) == 0, "block_size must be 16, 32, 64, 128 or 256, got " + std::to_string(bs));
    require_value(N > 0 && N < (1ll << 31) && H > 0 && H < (1ll << 24), "the cache must have blocks and heads");
    require_shape(c.k_scale, {N, H}, at::kFloat, c.k, "cache.k_scale");
    require_shape(c.v_scale, {N, H}, at::kFloat, c.k, "cache.v_scale");
    require_value(c.k_scale.is_contiguous() && c.v_scale.is_contiguous(), "cache.k_scale and cache.v_scale must be contiguous");
    corope_kv_cache_t r{};
    if (c.weight.has_value()) {
        require_shape(*c.weight, {N, H, bs}, at::kFloat, c.k, "cache.weight");
        require_value(c.weight->is_contiguous(), "cache.weight must be contiguous");
        r.weight = c.weight->data_ptr<float>();
    }
    for (const Tensor* t : {&c.k, &c.v}) {
        const auto st = t->strides();
        bool ok = st[3] == 1 && st[2] >= D && (uintptr_t)t->data_ptr() % 16 == 0;
        for (int i = 0; i < 3; ++i) ok = ok && st[i] >= 0 && st[i] % 16 == 0;
        require_value(ok, "rows of cache.k and cache.v must be contiguous and start at multiples of 16 bytes");
        require_value(!written || ((N == 1 || st[0] > 0) && (H == 1 || st[1] > 0)), "blocks and heads of cache.k and cache.v that are written to must not share memory");
    }
    r.k = c.k.data_ptr(); r.v = c.v.data_ptr();
    r.k_scale = c.k_scale.data_ptr<float>(); r.v_scale = c.v_scale.data_ptr<float>();
    set_strides(r.k_stride, c.k);
    set_strides(r.v_stride, c.v);
    r.num_blocks = (int)N; r.Hkv = (int)H; r.block_size = (int)bs; r.D = (int)D;
    r.code = c.k.scalar_type() == at::kChar ? COROPE_CODE_INT8 : COROPE_CODE_E4M3;
    return r;
}

const int* index_ptr(const Tensor& t, int64_t B, const Tensor& like, const char* name) {
    require_shape(t, {B}, at::kInt, like, name);
    require_value(t.is_contiguous(), std::string(name) + " must be contiguous");
    return t.data_ptr<int>();
}
void table_checks(const Tensor& t, int64_t B, const Tensor& like, const char* name) {
    require_cuda(t);
    require_value(t.dim() == 2 && t.size(0) == B && t.size(1) > 0 && t.size(1) < (1ll << 30) && t.scalar_type() == at::kInt && t.device() == like.device(),
                  std::string(name) + " must be an int32 tensor [B, blocks] on the cache's device");
    require_value((t.size(1) == 1 || t.stride(1) == 1) && (B == 1 || t.stride(0) >= t.size(1)), std::string(name) + " must have rows without gaps that do not overlap");
}
// `keep` holds what the tables were converted to
corope_cache_seqs_t seqs_view(const CacheTensors& c, const Tensor& block_table, const Tensor& seq_lens, const Optional& cos, const Optional& sin,
                              const Optional& positions, const Optional& new_lens, Tables& keep) {
    require_value(seq_lens.dim() == 1 && seq_lens.size(0) > 0 && seq_lens.size(0) < (1ll << 24), "seq_lens must be a tensor [B], of fewer than 2^24 sequences");
    const int64_t B = seq_lens.size(0), D = c.k.size(3);
    corope_cache_seqs_t r{};
    table_checks(block_table, B, c.k, "block_table");
    r.block_table = block_table.data_ptr<int>();
    r.table_stride = block_table.stride(0);
    r.B = (int)B;
    r.max_blocks = (int)block_table.size(1);
    r.seq_lens = index_ptr(seq_lens, B, c.k, "seq_lens");
    if (new_lens.has_value()) r.new_lens = index_ptr(*new_lens, B, c.k, "new_lens");
    if (positions.has_value()) r.positions = index_ptr(*positions, B, c.k, "positions");
    require_value(cos.has_value() == sin.has_value(), "give both freqs_cos and freqs_sin, or neither");
    if (cos.has_value()) {
        keep = tables(*cos, *sin, 1, D);
        require_value(keep.cos.device() == c.k.device() && keep.sin.device() == c.k.device(), "freqs_cos and freqs_sin must be on the cache's device");
        require_value(keep.cos.size(0) < (1ll << 31) && (keep.cos.size(0) == 1 || keep.stride >= D / 2), "rows of freqs_cos and freqs_sin must not overlap");
        r.cos = keep.cos.data_ptr<float>();
        r.sin = keep.sin.data_ptr<float>();
        r.rope_stride = keep.stride;
        r.table_rows = (int)keep.cos.size(0);
    }
    return r;
}
// rows as the cache kernels read them: any strides that are not negative, unit stride along the head dimension
Tensor readable_rows(const Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); }
void check_tokens(const Tensor& t, const CacheTensors& c, int64_t B, const char* name) {
    require_cuda(t);
    require_value(t.dim() == 4 && t.size(0) == B && t.size(2) > 0 && t.size(3) == c.k.size(3) && t.device() == c.k.device() && dtype_code(t) >= 0,
                  std::string(name) + " must be a [B, H, T, D] tensor in float32, bfloat16 or float16 with the cache's head dimension, on its device");
    require_value(t.size(2) <= (1 << 20), "at most 2^20 tokens a call");
}

void cache_append(const Tensor& k_in, const Tensor& v_in, const CacheTensors& c, const Tensor& block_table, const Tensor& seq_lens, const Optional& cos,
                  const Optional& sin, const Optional& positions, const Optional& new_lens) {
    require_no_grad({&k_in, &v_in}, c);
    const corope_kv_cache_t cache = cache_view(c, true);
    Call call(c.k);
    Tables keep;
    const corope_cache_seqs_t seqs = seqs_view(c, block_table, seq_lens, cos, sin, positions, new_lens, keep);
    check_tokens(k_in, c, seqs.B, "k");
    require_value(k_in.size(1) == cache.Hkv && k_in.sizes() == v_in.sizes() && k_in.scalar_type() == v_in.scalar_type() && v_in.device() == c.k.device(),
                  "k and v must share one shape, type and device and have the cache's heads");
    const Tensor k = readable_rows(k_in), v = readable_rows(v_in);
    int64_t sk[3], sv[3];
    set_strides(sk, k);
    set_strides(sv, v);
    raise_for_status(corope_cache_append(&cache, &seqs, k.data_ptr(), v.data_ptr(), sk, sv, (int)k.size(2), dtype_code(k), call.status.word_ptr, call.stream),
                     "corope_cache_append");
    whole_cache_written(c);
}

Tensor cache_attention(const Tensor& q_in, const CacheTensors& c, const Tensor& block_table, const Tensor& seq_lens, bool causal, double sm_scale,
                       const Optional& cos, const Optional& sin, const Optional& positions, const Optional& new_lens, bool accumulate) {
    require_no_grad({&q_in}, c);
    const corope_kv_cache_t cache = cache_view(c, false);
    Call call(c.k);
    Tables keep;
    const corope_cache_seqs_t seqs = seqs_view(c, block_table, seq_lens, cos, sin, positions, new_lens, keep);
    check_tokens(q_in, c, seqs.B, "q");
    require_value(q_in.size(1) > 0 && q_in.size(1) % cache.Hkv == 0, "Number of query heads must be divisible by KV heads.");
    require_value(!accumulate || cache.weight != nullptr, "accumulate needs a cache with weights");
    const Tensor q = readable_rows(q_in);
    // o is laid out like q, whose heads, tokens or batch entries may share memory; o's may not, and where q's overlap that can put the head dimension
    // somewhere else than last
    Tensor o = at::empty_like(q);
    if (o.stride(3) != 1) o = at::empty(q.sizes(), q.options());
    const int Hq = (int)q.size(1), T = (int)q.size(2), dt = dtype_code(q);
    const size_t bytes = corope_cache_attn_workspace_bytes(&cache, &seqs, Hq, T, dt, accumulate ? 1 : 0);
    const Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 256)}, q.options().dtype(at::kByte));
    int64_t sq[3], so[3];
    set_strides(sq, q);
    set_strides(so, o);
    raise_for_status(corope_cache_attn(&cache, &seqs, q.data_ptr(), o.data_ptr(), sq, so, Hq, T, dt, causal ? 1 : 0, (float)sm_scale, accumulate ? 1 : 0,
                                       ws.data_ptr(), bytes, call.status.word_ptr, call.stream),
                     "corope_cache_attn");
    if (accumulate) written({&*c.weight});
    return o;
}

std::tuple<Tensor, Tensor> cache_evict(const CacheTensors& c, const Tensor& block_table, const Tensor& seq_lens, const Tensor& out_table, int64_t budget,
                                       int64_t recent) {
    require_no_grad({}, c);
    const corope_kv_cache_t cache = cache_view(c, true);
    require_value(cache.weight != nullptr, "eviction needs a cache with weights");
    Call call(c.k);
    Tables keep;
    const corope_cache_seqs_t seqs = seqs_view(c, block_table, seq_lens, {}, {}, {}, {}, keep);
    table_checks(out_table, seqs.B, c.k, "out_table");
    require_value(budget > 0 && budget < (1ll << 30) && recent >= 0 && recent <= budget, "budget must be positive (below 2^30) and recent between 0 and budget");
    require_value(out_table.size(1) * cache.block_size >= budget, "out_table's blocks must hold budget tokens");
    const auto ints = seq_lens.options();
    Tensor lens = at::empty({seqs.B}, ints), kept = at::empty({seqs.B, cache.Hkv, budget}, ints);
    raise_for_status(corope_cache_evict(&cache, &seqs, out_table.data_ptr<int>(), out_table.stride(0), (int)out_table.size(1), (int)budget, (int)recent,
                                        lens.data_ptr<int>(), kept.data_ptr<int>(), call.status.word_ptr, call.stream),
                     "corope_cache_evict");
    whole_cache_written(c);
    return {lens, kept};
}

// ------------------------------------------------------------------------------------------------ autograd nodes
Tensor save(AutogradContext* ctx, Kind kind, const Saved& s, bool causal, double sm_scale, double theta) {
    variable_list t{s.q, s.k, s.v, s.o, s.m};
    if (kind == kRope) t.insert(t.end(), {s.tab.cos, s.tab.sin});
    ctx->save_for_backward(std::move(t));
    ctx->saved_data["kind"] = (int64_t)kind;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["sm_scale"] = sm_scale;
    ctx->saved_data["theta"] = theta;
    return s.o;
}
Grads saved_backward(AutogradContext* ctx, const Tensor& d_out) {
    const variable_list t = ctx->get_saved_variables();
    const Kind kind = (Kind)ctx->saved_data["kind"].toInt();
    Saved s{t[0], t[1], t[2], t[3], t[4], {}};
    if (kind == kRope) s.tab = Tables{t[5], t[6], t[5].stride(0)};
    return mha_backward(kind, s, d_out, ctx->saved_data["causal"].toBool(), ctx->saved_data["sm_scale"].toDouble(), ctx->saved_data["theta"].toDouble());
}

struct RopeFunction : torch::autograd::Function<RopeFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, const Tensor& cos,
                          const Tensor& sin) {
        return save(ctx, kRope, mha_forward(kRope, q, k, v, causal, sm_scale, cos, sin, 0.0), causal, sm_scale, 0.0);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        Grads g = saved_backward(ctx, grads[0]);
        return {g.dq, g.dk, g.dv, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct MhaFunction : torch::autograd::Function<MhaFunction> {   // without table arguments
    static Tensor forward(AutogradContext* ctx, int64_t kind, const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, double theta) {
        return save(ctx, (Kind)kind, mha_forward((Kind)kind, q, k, v, causal, sm_scale, Tensor(), Tensor(), theta), causal, sm_scale, theta);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        Grads g = saved_backward(ctx, grads[0]);
        return {Tensor(), g.dq, g.dk, g.dv, Tensor(), Tensor(), Tensor()};
    }
};

struct GqaFunction : torch::autograd::Function<GqaFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, double theta) {
        GqaSaved s = gqa_forward(q, k, v, causal, sm_scale, theta);
        ctx->save_for_backward({s.q, s.k, s.v, s.o, s.lse2, s.a_diag});
        ctx->saved_data["sm_scale"] = sm_scale;
        ctx->saved_data["theta"] = theta;
        return s.o;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list t = ctx->get_saved_variables();
        Grads g = gqa_backward(GqaSaved{t[0], t[1], t[2], t[3], t[4], t[5]}, grads[0], ctx->saved_data["sm_scale"].toDouble(),
                               ctx->saved_data["theta"].toDouble());
        return {g.dq, g.dk, g.dv, Tensor(), Tensor(), Tensor()};
    }
};

}  // namespace

PYBIND11_MODULE(_corope_torch, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const AssertError& e) {
            PyErr_SetString(PyExc_AssertionError, e.what());
        } catch (const ValueError& e) {
            PyErr_SetString(PyExc_ValueError, e.what());
        }
    });
    // The GIL is released for every call: a launch blocks once the launch queue is full, and other Python threads go on meanwhile.
    // autograd entry points
    using NoGil = py::call_guard<py::gil_scoped_release>;
    m.def("rope_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, const Tensor& cos, const Tensor& sin) {
        return RopeFunction::apply(q, k, v, causal, sm_scale, cos, sin);
    }, NoGil());
    m.def("theta_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, double theta) {
        return MhaFunction::apply((int64_t)kTheta, q, k, v, causal, sm_scale, theta);
    }, NoGil());
    m.def("flash_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale) {
        return MhaFunction::apply((int64_t)kFlash, q, k, v, causal, sm_scale, 0.0);
    }, NoGil());
    m.def("gqa_attention", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, double theta) {
        return GqaFunction::apply(q, k, v, causal, sm_scale, theta);
    }, NoGil());
    // the library calls alone, without autograd
    m.def("rope_forward", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, const Tensor& cos, const Tensor& sin) {
        Saved s = mha_forward(kRope, q, k, v, causal, sm_scale, cos, sin, 0.0);
        return std::make_tuple(s.q, s.k, s.v, s.o, s.m, s.tab.cos, s.tab.sin, s.tab.stride);
    }, NoGil());
    m.def("rope_backward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& cos, const Tensor& sin,
                              int64_t stride, const Tensor& d_o, bool causal, double sm_scale) {
        Grads g = mha_backward(kRope, Saved{q, k, v, o, lse, Tables{cos, sin, stride}}, d_o, causal, sm_scale, 0.0);
        return std::make_tuple(g.dq, g.dk, g.dv);
    }, NoGil());
    m.def("gqa_forward", [](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double sm_scale, double theta) {
        GqaSaved s = gqa_forward(q, k, v, causal, sm_scale, theta);
        return std::make_tuple(s.q, s.k, s.v, s.o, s.lse2, s.a_diag);
    }, NoGil());
    m.def("gqa_backward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse2, const Tensor& a_diag, const Tensor& d_o,
                             double sm_scale, double theta) {
        Grads g = gqa_backward(GqaSaved{q, k, v, o, lse2, a_diag}, d_o, sm_scale, theta);
        return std::make_tuple(g.dq, g.dk, g.dv);
    }, NoGil());
    // the 8-bit cache: (k, v, k_scale, v_scale, weight) stand for the cache object
    m.def("cache_append", [](const Tensor& k, const Tensor& v, const Tensor& ck, const Tensor& cv, const Tensor& ks, const Tensor& vs, const Optional& w,
                             const Tensor& table, const Tensor& lens, const Optional& cos, const Optional& sin, const Optional& positions, const Optional& new_lens) {
        cache_append(k, v, CacheTensors{ck, cv, ks, vs, w}, table, lens, cos, sin, positions, new_lens);
    }, NoGil());
    m.def("cache_attention", [](const Tensor& q, const Tensor& ck, const Tensor& cv, const Tensor& ks, const Tensor& vs, const Optional& w, const Tensor& table,
                                const Tensor& lens, bool causal, double sm_scale, const Optional& cos, const Optional& sin, const Optional& positions,
                                const Optional& new_lens, bool accumulate) {
        return cache_attention(q, CacheTensors{ck, cv, ks, vs, w}, table, lens, causal, sm_scale, cos, sin, positions, new_lens, accumulate);
    }, NoGil());
    m.def("cache_evict", [](const Tensor& ck, const Tensor& cv, const Tensor& ks, const Tensor& vs, const Optional& w, const Tensor& table, const Tensor& lens,
                            const Tensor& out_table, int64_t budget, int64_t recent) {
        return cache_evict(CacheTensors{ck, cv, ks, vs, w}, table, lens, out_table, budget, recent);
    }, NoGil());
    // (status word tensor, pinned mirror tensor) of a device, created on first use
    m.def("device_status", [](int index) {
        c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
        DeviceStatus& st = device_status(index);
        return std::make_tuple(st.word, st.mirror);
    }, NoGil());
}
