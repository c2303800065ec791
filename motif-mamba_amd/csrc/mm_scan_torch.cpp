// mm_scan_torch.cpp -- thin PyTorch-ROCm binding over the C ABI of libmm_scan.so.
//
// fwd(...)        mirrors selective_scan_cuda.fwd (reference csrc/selective_scan/selective_scan.cpp:
//                 270-413, pybind :620-627): same argument names, checks and outputs
//                 [out, x, out_z?], where x is the (batch, dim, ceil(L/2048), 2*dstate) float32
//                 chunk-state tensor of interleaved (prod a, h) pairs.
// fwd_infer(...)  the inference form used by SelectiveScanFn: writes only the returned output
//                 (out_z when z is given, else out) and, on request, a contiguous last_state.
// state_update(.) the decode step (replaces upstream selective_state_update, called at
//                 mamba_ssm/modules/mamba_simplemotif.py:397-399).
// Validation failures raise RuntimeError through TORCH_CHECK, like the reference binding.
// ROCm torch reports GPU tensors with device type "cuda"; the generic c10::DeviceGuard accepts it,
// and c10::hip::getCurrentHIPStream() is the stream torch launches its own HIP work on.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdlib>
#include <vector>

#include "mm_conv1d.h"
#include "mm_delta.h"
#include "mm_group_norm.h"
#include "mm_layer_norm.h"
#include "mm_linattn.h"
#include "mm_norm.h"
#include "mm_scan.h"

namespace {

#define CHECK_SHAPE(x, ...) \
    TORCH_CHECK(x.sizes() == torch::IntArrayRef({__VA_ARGS__}), #x " must have shape (" #__VA_ARGS__ ")")

mm_dtype to_mm(at::ScalarType t) {
    switch (t) {
        case at::ScalarType::Float: return MM_FLOAT32;
        case at::ScalarType::Half: return MM_FLOAT16;
        case at::ScalarType::BFloat16: return MM_BFLOAT16;
        default: AT_ERROR("selective_scan_fwd not implemented for input type '", c10::toString(t), "'");
    }
}

void check_rc(int rc, const char *what) {
    if (rc == MM_ERR_UNSUPPORTED) {
        // A shape the kernels do not cover: NotImplementedError (a RuntimeError) in Python.
        throw c10::NotImplementedError({__func__, __FILE__, uint32_t(__LINE__)},
                                       c10::str(what, " failed (code ", rc, "): ", mm_last_error()));
    }
    TORCH_CHECK(rc == MM_OK, what, " failed (code ", rc, "): ", mm_last_error());
}

struct FwdSetup {
    mm_scan_fwd_params p;
    int64_t n_chunks;
};

// Shared validation (selective_scan.cpp:280-381, without the P/Q/gamma and complex branches,
// which attach_pq and the complex-A refusal below cover).
FwdSetup setup_fwd(const at::Tensor &u, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B,
                   const at::Tensor &C, const c10::optional<at::Tensor> &D_, const c10::optional<at::Tensor> &z_,
                   const c10::optional<at::Tensor> &delta_bias_, bool delta_softplus) {
    const auto input_type = u.scalar_type();
    const auto weight_type = A.scalar_type();
    TORCH_CHECK(input_type == at::ScalarType::Float || input_type == at::ScalarType::Half ||
                input_type == at::ScalarType::BFloat16);
    TORCH_CHECK(weight_type == at::ScalarType::Float || weight_type == at::ScalarType::ComplexFloat);
    if (weight_type == at::ScalarType::ComplexFloat) {
        throw c10::NotImplementedError({__func__, __FILE__, uint32_t(__LINE__)},
                                       "complex A is not supported by the MI355X selective scan");
    }
    const bool is_variable_B = B.dim() >= 3;
    const bool is_variable_C = C.dim() >= 3;
    TORCH_CHECK(delta.scalar_type() == input_type);
    TORCH_CHECK(B.scalar_type() == (!is_variable_B ? weight_type : input_type));
    TORCH_CHECK(C.scalar_type() == (!is_variable_C ? weight_type : input_type));
    TORCH_CHECK(u.is_cuda());
    TORCH_CHECK(delta.is_cuda());
    TORCH_CHECK(A.is_cuda());
    TORCH_CHECK(B.is_cuda());
    TORCH_CHECK(C.is_cuda());
    TORCH_CHECK(u.stride(-1) == 1 || u.size(-1) == 1);
    TORCH_CHECK(delta.stride(-1) == 1 || delta.size(-1) == 1);

    TORCH_CHECK(u.dim() == 3, "u must have shape (batch, dim, seqlen)");
    const int64_t batch_size = u.size(0), dim = u.size(1), seqlen = u.size(2);
    TORCH_CHECK(A.dim() == 2, "A must have shape (dim, dstate)");
    const int64_t dstate = A.size(1);
    TORCH_CHECK(!is_variable_B || B.dim() == 4, "variable B must be 4-D (batch, n_groups, dstate, seqlen)");
    const int64_t n_groups = is_variable_B ? B.size(1) : 1;
    TORCH_CHECK(dstate <= MM_SCAN_MAX_DSTATE, "selective_scan only supports state dimension <= 256");

    CHECK_SHAPE(u, batch_size, dim, seqlen);
    CHECK_SHAPE(delta, batch_size, dim, seqlen);
    CHECK_SHAPE(A, dim, dstate);
    if (!is_variable_B) {
        CHECK_SHAPE(B, dim, dstate);
    } else {
        CHECK_SHAPE(B, batch_size, n_groups, dstate, seqlen);
        TORCH_CHECK(B.stride(-1) == 1 || B.size(-1) == 1);
    }
    if (!is_variable_C) {
        CHECK_SHAPE(C, dim, dstate);
    } else {
        TORCH_CHECK(C.dim() == 4, "variable C must be 4-D (batch, n_groups, dstate, seqlen)");
        CHECK_SHAPE(C, batch_size, n_groups, dstate, seqlen);
        TORCH_CHECK(C.stride(-1) == 1 || C.size(-1) == 1);
    }
    TORCH_CHECK(n_groups >= 1 && dim % n_groups == 0, "dim must be a multiple of n_groups");
    if (D_.has_value()) {
        const auto &D = D_.value();
        TORCH_CHECK(D.scalar_type() == at::ScalarType::Float);
        TORCH_CHECK(D.is_cuda());
        TORCH_CHECK(D.stride(-1) == 1 || D.size(-1) == 1);
        CHECK_SHAPE(D, dim);
    }
    if (delta_bias_.has_value()) {
        const auto &db = delta_bias_.value();
        TORCH_CHECK(db.scalar_type() == at::ScalarType::Float);
        TORCH_CHECK(db.is_cuda());
        TORCH_CHECK(db.stride(-1) == 1 || db.size(-1) == 1);
        CHECK_SHAPE(db, dim);
    }
    if (z_.has_value()) {
        const auto &z = z_.value();
        TORCH_CHECK(z.scalar_type() == input_type);
        TORCH_CHECK(z.is_cuda());
        TORCH_CHECK(z.stride(-1) == 1 || z.size(-1) == 1);
        CHECK_SHAPE(z, batch_size, dim, seqlen);
    }

    FwdSetup s;
    std::memset(&s.p, 0, sizeof(s.p));
    mm_scan_fwd_params &p = s.p;
    p.batch = batch_size;
    p.dim = dim;
    p.seqlen = seqlen;
    p.dstate = dstate;
    p.n_groups = n_groups;
    p.itype = to_mm(input_type);
    p.is_variable_B = is_variable_B;
    p.is_variable_C = is_variable_C;
    p.delta_softplus = delta_softplus;
    p.u = u.data_ptr();
    p.delta = delta.data_ptr();
    p.A = A.data_ptr<float>();
    p.B = B.data_ptr();
    p.C = C.data_ptr();
    p.D = D_.has_value() ? D_.value().data_ptr<float>() : nullptr;
    p.z = z_.has_value() ? z_.value().data_ptr() : nullptr;
    p.delta_bias = delta_bias_.has_value() ? delta_bias_.value().data_ptr<float>() : nullptr;
    p.u_batch_stride = u.stride(0);
    p.u_d_stride = u.stride(1);
    p.delta_batch_stride = delta.stride(0);
    p.delta_d_stride = delta.stride(1);
    if (z_.has_value()) {
        p.z_batch_stride = z_.value().stride(0);
        p.z_d_stride = z_.value().stride(1);
    }
    p.A_d_stride = A.stride(0);
    p.A_dstate_stride = A.stride(1);
    if (is_variable_B) {
        p.B_batch_stride = B.stride(0);
        p.B_group_stride = B.stride(1);
        p.B_dstate_stride = B.stride(2);
    } else {
        p.B_d_stride = B.stride(0);
        p.B_dstate_stride = B.stride(1);
    }
    if (is_variable_C) {
        p.C_batch_stride = C.stride(0);
        p.C_group_stride = C.stride(1);
        p.C_dstate_stride = C.stride(2);
    } else {
        p.C_d_stride = C.stride(0);
        p.C_dstate_stride = C.stride(1);
    }
    s.n_chunks = (seqlen + MM_SCAN_CHUNK - 1) / MM_SCAN_CHUNK;
    return s;
}

void set_out(mm_scan_fwd_params &p, const at::Tensor &out) {
    p.out = out.data_ptr();
    p.out_batch_stride = out.stride(0);
    p.out_d_stride = out.stride(1);
}

void set_out_z(mm_scan_fwd_params &p, const at::Tensor &out_z) {
    p.out_z = out_z.data_ptr();
    p.out_z_batch_stride = out_z.stride(0);
    p.out_z_d_stride = out_z.stride(1);
}

// Low-rank coupling P/Q and gamma (checks of selective_scan.cpp:342-369, strides as
// set_ssm_params_fwd, selective_scan.cpp:149-164). P and Q are read as float32: the reference's
// dense kernel reinterprets them as float and its full-matrix path upcasts them with .float().
// gamma is validated and carried, not read (neither reference forward reads it). Returns the
// float32 P/Q the parameter block points at; the caller keeps them alive until the launch.
std::vector<at::Tensor> attach_pq(mm_scan_fwd_params &p, const at::Tensor &u, const c10::optional<at::Tensor> &P_,
                                  const c10::optional<at::Tensor> &Q_, const c10::optional<at::Tensor> &gamma_) {
    TORCH_CHECK(!P_.has_value() || Q_.has_value(), "Q must be provided when P is provided");
    TORCH_CHECK(!Q_.has_value() || P_.has_value(), "P must be provided when Q is provided");
    std::vector<at::Tensor> keep;
    if (P_.has_value()) {
        const at::Tensor &P = P_.value(), &Q = Q_.value();
        TORCH_CHECK(P.is_cuda() && Q.is_cuda(), "P and Q must be CUDA tensors");
        TORCH_CHECK(P.device() == u.device() && Q.device() == u.device(), "P and Q must be on the device of u");
        TORCH_CHECK(P.dim() == Q.dim() && (P.dim() == 2 || P.dim() == 3), "P/Q must be 2D or 3D with same rank");
        if (P.dim() == 2) {
            TORCH_CHECK(P.size(0) == p.dstate && Q.size(1) == p.dstate && P.size(1) == Q.size(0),
                        "Expect P(dstate, r), Q(r, dstate)");
        } else {
            TORCH_CHECK(P.size(0) == p.dim && Q.size(0) == p.dim, "P/Q dim mismatch");
            TORCH_CHECK(P.size(1) == p.dstate && Q.size(2) == p.dstate && P.size(2) == Q.size(1),
                        "Expect P(dim, dstate, r), Q(dim, r, dstate)");
        }
        TORCH_CHECK(P.size(-1) <= 8, "Current dense CUDA forward supports pq_rank <= 8");
        const at::Tensor Pf = P.to(at::ScalarType::Float), Qf = Q.to(at::ScalarType::Float);
        keep = {Pf, Qf};
        p.P = Pf.data_ptr<float>();
        p.Q = Qf.data_ptr<float>();
        p.pq_rank = P.size(-1);
        p.P_d_stride = P.dim() == 3 ? Pf.stride(0) : 0;
        p.P_dstate_stride = Pf.stride(P.dim() - 2);
        p.P_r_stride = Pf.stride(P.dim() - 1);
        p.Q_d_stride = Q.dim() == 3 ? Qf.stride(0) : 0;
        p.Q_r_stride = Qf.stride(Q.dim() - 2);
        p.Q_dstate_stride = Qf.stride(Q.dim() - 1);
    }
    if (gamma_.has_value()) {
        const at::Tensor &gamma = gamma_.value();
        TORCH_CHECK(gamma.is_cuda(), "gamma must be CUDA tensor");
        TORCH_CHECK(gamma.dim() == 1 || gamma.dim() == 2, "gamma must be 1D or 2D");
        if (gamma.dim() == 1) {
            TORCH_CHECK(gamma.size(0) == p.dstate, "gamma(1D) shape must be (dstate,)");
        } else {
            TORCH_CHECK(gamma.size(0) == p.dim && gamma.size(1) == p.dstate, "gamma(2D) shape must be (dim, dstate)");
        }
        p.gamma = static_cast<const float *>(gamma.data_ptr());
        p.gamma_d_stride = gamma.dim() == 2 ? gamma.stride(0) : 0;
        p.gamma_dstate_stride = gamma.stride(-1);
    }
    return keep;
}

// Scratch for the sequence-parallel segments (only for shapes that use them), from the caching
// allocator on the launch stream: released when the caller's reference drops, stream-ordered.
at::Tensor attach_workspace(mm_scan_fwd_params &p, const at::Tensor &like) {
    const int64_t bytes = mm_scan_fwd_workspace_size(&p);
    if (bytes <= 0) return at::Tensor();
    at::Tensor ws = torch::empty({bytes}, like.options().dtype(at::ScalarType::Byte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = bytes;
    return ws;
}

std::vector<at::Tensor> fwd(const at::Tensor &u, const at::Tensor &delta, const at::Tensor &A,
                            const at::Tensor &B, const at::Tensor &C, const c10::optional<at::Tensor> &D_,
                            const c10::optional<at::Tensor> &z_, const c10::optional<at::Tensor> &delta_bias_,
                            const c10::optional<at::Tensor> &P_, const c10::optional<at::Tensor> &Q_,
                            const c10::optional<at::Tensor> &gamma_, bool delta_softplus, bool tile_states) {
    FwdSetup s = setup_fwd(u, delta, A, B, C, D_, z_, delta_bias_, delta_softplus);
    mm_scan_fwd_params &p = s.p;
    const std::vector<at::Tensor> pq = attach_pq(p, u, P_, Q_, gamma_);
    // Output layouts follow the reference: out like delta, out_z like z (like out when z is a
    // non-dense view such as half of xz), x contiguous.
    at::Tensor out = torch::empty_like(delta);
    at::Tensor x = torch::empty({p.batch, p.dim, s.n_chunks, p.dstate * 2}, u.options().dtype(A.scalar_type()));
    at::Tensor out_z;
    set_out(p, out);
    if (z_.has_value()) {
        out_z = z_.value().is_non_overlapping_and_dense() ? torch::empty_like(z_.value()) : torch::empty_like(out);
        set_out_z(p, out_z);
    }
    p.chunk_states = x.data_ptr<float>();
    // tile_states (this build's addition): the states before every 16-step tile, appended to the
    // outputs for the backward -- None when the kernels cannot write them for this request (the
    // query sees the final parameter block, outputs included).
    at::Tensor ck;
    if (tile_states && mm_scan_fwd_tile_states_size(&p) > 0) {
        ck = torch::empty({(p.seqlen + 15) / 16, p.batch, p.dim, 16}, u.options().dtype(at::ScalarType::Float));
        p.tile_states = ck.data_ptr<float>();
    }
    const c10::DeviceGuard device_guard{u.device()};
    const at::Tensor ws = attach_workspace(p, u);
    check_rc(mm_scan_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_scan_fwd");
    std::vector<at::Tensor> result = {out, x};
    if (z_.has_value()) result.push_back(out_z);
    if (tile_states) result.push_back(ck);
    return result;
}

std::vector<at::Tensor> fwd_infer(const at::Tensor &u, const at::Tensor &delta, const at::Tensor &A,
                                  const at::Tensor &B, const at::Tensor &C, const c10::optional<at::Tensor> &D_,
                                  const c10::optional<at::Tensor> &z_,
                                  const c10::optional<at::Tensor> &delta_bias_, bool delta_softplus,
                                  bool return_last_state, const c10::optional<at::Tensor> &P_,
                                  const c10::optional<at::Tensor> &Q_, const c10::optional<at::Tensor> &gamma_) {
    FwdSetup s = setup_fwd(u, delta, A, B, C, D_, z_, delta_bias_, delta_softplus);
    mm_scan_fwd_params &p = s.p;
    const std::vector<at::Tensor> pq = attach_pq(p, u, P_, Q_, gamma_);
    at::Tensor main;
    if (z_.has_value()) {
        main = z_.value().is_non_overlapping_and_dense() ? torch::empty_like(z_.value()) : torch::empty_like(delta);
        set_out_z(p, main);
    } else {
        main = torch::empty_like(delta);
        set_out(p, main);
    }
    at::Tensor last_state;
    if (return_last_state) {
        last_state = torch::empty({p.batch, p.dim, p.dstate}, u.options().dtype(at::ScalarType::Float));
        p.last_state = last_state.data_ptr<float>();
    }
    const c10::DeviceGuard device_guard{u.device()};
    const at::Tensor ws = attach_workspace(p, u);
    check_rc(mm_scan_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_scan_fwd");
    if (return_last_state) return {main, last_state};
    return {main};
}


// selective_scan_cuda.bwd (selective_scan.cpp:415-612): [du, ddelta, dA, dB, dC, dD, ddelta_bias,
// dz?, out_z?]. x (the forward's chunk states) is checked like the reference but not read: the
// backward recomputes the forward states itself. With P/Q the exact gradient of the coupled
// recurrence runs (pq_rank 1..8, any dstate up to 256).
std::vector<at::Tensor> bwd(const at::Tensor &u, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B,
                            const at::Tensor &C, const c10::optional<at::Tensor> &D_,
                            const c10::optional<at::Tensor> &z_, const c10::optional<at::Tensor> &delta_bias_,
                            const c10::optional<at::Tensor> &P_, const c10::optional<at::Tensor> &Q_,
                            const c10::optional<at::Tensor> &gamma_, const at::Tensor &dout,
                            const c10::optional<at::Tensor> &x_, const c10::optional<at::Tensor> &out_,
                            c10::optional<at::Tensor> dz_, const c10::optional<at::Tensor> &dP_out_,
                            const c10::optional<at::Tensor> &dQ_out_, bool delta_softplus, bool recompute_out_z,
                            const c10::optional<at::Tensor> &tile_states_) {
    FwdSetup s = setup_fwd(u, delta, A, B, C, D_, z_, delta_bias_, delta_softplus);
    // P/Q (and gamma, validated and not read, as in the forward): the float32 copies stay alive
    // until the launch is enqueued.
    const std::vector<at::Tensor> pq_keep = attach_pq(s.p, u, P_, Q_, gamma_);
    const mm_scan_fwd_params &f = s.p;
    // Rank-0 P/Q couple nothing: their forward is the diagonal scan and so is the backward (dP and
    // dQ are empty).
    const bool has_pq = P_.has_value() && f.pq_rank > 0;
    TORCH_CHECK(P_.has_value() || (!dP_out_.has_value() && !dQ_out_.has_value()), "dP_out and dQ_out need P and Q");
    (void)pq_keep;
    TORCH_CHECK(dout.scalar_type() == u.scalar_type());
    TORCH_CHECK(dout.is_cuda());
    TORCH_CHECK(dout.stride(-1) == 1 || dout.size(-1) == 1);
    CHECK_SHAPE(dout, f.batch, f.dim, f.seqlen);
    at::Tensor out, dz, out_z;
    const bool has_z = z_.has_value();
    if (has_z) {
        TORCH_CHECK(out_.has_value());
        out = out_.value();
        TORCH_CHECK(out.scalar_type() == u.scalar_type());
        TORCH_CHECK(out.is_cuda());
        TORCH_CHECK(out.stride(-1) == 1 || out.size(-1) == 1);
        CHECK_SHAPE(out, f.batch, f.dim, f.seqlen);
        if (dz_.has_value()) {
            dz = dz_.value();
            TORCH_CHECK(dz.scalar_type() == u.scalar_type());
            TORCH_CHECK(dz.is_cuda());
            TORCH_CHECK(dz.stride(-1) == 1 || dz.size(-1) == 1);
            CHECK_SHAPE(dz, f.batch, f.dim, f.seqlen);
        } else {
            dz = torch::empty_like(z_.value());
        }
        if (recompute_out_z) out_z = torch::empty_like(out);
    }
    if (s.n_chunks > 1) TORCH_CHECK(x_.has_value());
    if (x_.has_value()) {
        const at::Tensor &x = x_.value();
        TORCH_CHECK(x.scalar_type() == A.scalar_type());
        TORCH_CHECK(x.is_cuda());
        TORCH_CHECK(x.is_contiguous());
        CHECK_SHAPE(x, f.batch, f.dim, s.n_chunks, 2 * f.dstate);
    }
    at::Tensor du = torch::empty_like(u);
    at::Tensor ddelta = torch::empty_like(delta);
    at::Tensor dA = torch::empty_like(A);
    at::Tensor dB = torch::empty(B.sizes(), B.options().dtype(at::ScalarType::Float));
    at::Tensor dC = torch::empty(C.sizes(), C.options().dtype(at::ScalarType::Float));
    at::Tensor dD, ddelta_bias;
    if (D_.has_value()) dD = torch::empty_like(D_.value());
    if (delta_bias_.has_value()) ddelta_bias = torch::empty_like(delta_bias_.value());

    mm_scan_bwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = f.batch; p.dim = f.dim; p.seqlen = f.seqlen; p.dstate = f.dstate; p.n_groups = f.n_groups;
    p.itype = f.itype; p.is_variable_B = f.is_variable_B; p.is_variable_C = f.is_variable_C;
    p.delta_softplus = f.delta_softplus;
    p.u = f.u; p.delta = f.delta; p.A = f.A; p.B = f.B; p.C = f.C; p.D = f.D; p.z = f.z; p.delta_bias = f.delta_bias;
    p.u_batch_stride = f.u_batch_stride; p.u_d_stride = f.u_d_stride;
    p.delta_batch_stride = f.delta_batch_stride; p.delta_d_stride = f.delta_d_stride;
    p.z_batch_stride = f.z_batch_stride; p.z_d_stride = f.z_d_stride;
    p.A_d_stride = f.A_d_stride; p.A_dstate_stride = f.A_dstate_stride;
    p.B_batch_stride = f.B_batch_stride; p.B_group_stride = f.B_group_stride;
    p.B_dstate_stride = f.B_dstate_stride; p.B_d_stride = f.B_d_stride;
    p.C_batch_stride = f.C_batch_stride; p.C_group_stride = f.C_group_stride;
    p.C_dstate_stride = f.C_dstate_stride; p.C_d_stride = f.C_d_stride;
    p.dout = dout.data_ptr();
    p.dout_batch_stride = dout.stride(0); p.dout_d_stride = dout.stride(1);
    if (has_z) {
        p.out = out.data_ptr(); p.out_batch_stride = out.stride(0); p.out_d_stride = out.stride(1);
        p.dz = dz.data_ptr(); p.dz_batch_stride = dz.stride(0); p.dz_d_stride = dz.stride(1);
        if (recompute_out_z) {
            p.out_z = out_z.data_ptr(); p.out_z_batch_stride = out_z.stride(0); p.out_z_d_stride = out_z.stride(1);
        }
    }
    p.du = du.data_ptr(); p.du_batch_stride = du.stride(0); p.du_d_stride = du.stride(1);
    p.ddelta = ddelta.data_ptr(); p.ddelta_batch_stride = ddelta.stride(0); p.ddelta_d_stride = ddelta.stride(1);
    p.dA = dA.data_ptr<float>(); p.dA_d_stride = dA.stride(0); p.dA_dstate_stride = dA.stride(1);
    p.dB = dB.data_ptr<float>();
    p.dC = dC.data_ptr<float>();
    if (f.is_variable_B) {
        p.dB_batch_stride = dB.stride(0); p.dB_group_stride = dB.stride(1); p.dB_dstate_stride = dB.stride(2);
    } else {
        p.dB_d_stride = dB.stride(0); p.dB_dstate_stride = dB.stride(1);
    }
    if (f.is_variable_C) {
        p.dC_batch_stride = dC.stride(0); p.dC_group_stride = dC.stride(1); p.dC_dstate_stride = dC.stride(2);
    } else {
        p.dC_d_stride = dC.stride(0); p.dC_dstate_stride = dC.stride(1);
    }
    if (D_.has_value()) p.dD = dD.data_ptr<float>();
    if (delta_bias_.has_value()) p.ddelta_bias = ddelta_bias.data_ptr<float>();
    // dP / dQ (selective_scan.cpp:580-590): the exact gradients of the coupled recurrence are
    // added into dP_out / dQ_out (float32, the shapes of P and Q) when given, as the reference
    // accumulates into them; without them they are computed and dropped, as there, and the
    // result list is the reference's either way.
    at::Tensor dP, dQ;
    if (has_pq) {
        const at::Tensor &P = P_.value(), &Q = Q_.value();
        if (dP_out_.has_value() || dQ_out_.has_value()) {
            TORCH_CHECK(dP_out_.has_value() && dQ_out_.has_value(), "dP_out and dQ_out go together");
            const at::Tensor &dPo = dP_out_.value(), &dQo = dQ_out_.value();
            TORCH_CHECK(dPo.is_cuda() && dQo.is_cuda(), "dP_out and dQ_out must be CUDA tensors");
            TORCH_CHECK(dPo.scalar_type() == at::ScalarType::Float && dQo.scalar_type() == at::ScalarType::Float,
                        "dP_out and dQ_out must be float32");
            TORCH_CHECK(dPo.sizes() == P.sizes(), "dP_out shape mismatch");
            TORCH_CHECK(dQo.sizes() == Q.sizes(), "dQ_out shape mismatch");
        }
        dP = torch::empty(P.sizes(), P.options().dtype(at::ScalarType::Float));
        dQ = torch::empty(Q.sizes(), Q.options().dtype(at::ScalarType::Float));
        p.P = f.P; p.Q = f.Q; p.pq_rank = f.pq_rank;
        p.P_d_stride = f.P_d_stride; p.P_dstate_stride = f.P_dstate_stride; p.P_r_stride = f.P_r_stride;
        p.Q_d_stride = f.Q_d_stride; p.Q_r_stride = f.Q_r_stride; p.Q_dstate_stride = f.Q_dstate_stride;
        p.dP = dP.data_ptr<float>();
        p.dQ = dQ.data_ptr<float>();
        p.dP_d_stride = P.dim() == 3 ? dP.stride(0) : 0;
        p.dP_dstate_stride = dP.stride(P.dim() - 2);
        p.dP_r_stride = dP.stride(P.dim() - 1);
        p.dQ_d_stride = Q.dim() == 3 ? dQ.stride(0) : 0;
        p.dQ_r_stride = dQ.stride(Q.dim() - 2);
        p.dQ_dstate_stride = dQ.stride(Q.dim() - 1);
    }
    if (tile_states_.has_value()) {
        const at::Tensor &ck = tile_states_.value();
        TORCH_CHECK(ck.is_cuda() && ck.scalar_type() == at::ScalarType::Float && ck.is_contiguous() &&
                        ck.sizes() == at::IntArrayRef({(f.seqlen + 15) / 16, f.batch, f.dim, 16}),
                    "tile_states must be the contiguous float32 (ceil(L / 16), batch, dim, 16) tensor of the forward");
        p.tile_states = ck.data_ptr<float>();
    }
    const c10::DeviceGuard device_guard{u.device()};
    at::Tensor ws;
    const int64_t ws_bytes = mm_scan_bwd_workspace_size(&p);
    if (ws_bytes > 0) {
        ws = torch::empty({ws_bytes}, u.options().dtype(at::ScalarType::Byte));
        p.workspace = ws.data_ptr();
        p.workspace_bytes = ws_bytes;
    }
    check_rc(mm_scan_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_scan_bwd");
    std::vector<at::Tensor> result = {du, ddelta, dA, dB.to(B.scalar_type()), dC.to(C.scalar_type()), dD, ddelta_bias};
    if (has_z) result.push_back(dz);
    if (recompute_out_z) result.push_back(out_z);
    if (has_pq && dP_out_.has_value()) {
        dP_out_.value().add_(dP);
        dQ_out_.value().add_(dQ);
    }
    return result;
}


mm_dtype conv_dtype(const at::Tensor &t, const char *what) {
    const auto st = t.scalar_type();
    TORCH_CHECK(st == at::ScalarType::Float || st == at::ScalarType::Half || st == at::ScalarType::BFloat16,
                what, " must be float32, float16 or bfloat16");
    return to_mm(st);
}

// causal_conv1d_fwd (package causal-conv1d; fallback mamba_simplemotif.py:298-299): out (written into
// `out` when given, in any layout contiguous along seqlen), and the last width - 1 inputs into
// final_states_out when given.
at::Tensor conv1d_fwd(const at::Tensor &x, const at::Tensor &weight, const c10::optional<at::Tensor> &bias_,
                      const c10::optional<at::Tensor> &initial_states_, const c10::optional<at::Tensor> &final_states_out_,
                      bool silu, const c10::optional<at::Tensor> &out_) {
    TORCH_CHECK(x.is_cuda() && weight.is_cuda(), "x and weight must be on the GPU");
    TORCH_CHECK(x.dim() == 3, "x must have shape (batch, dim, seqlen)");
    TORCH_CHECK(x.stride(-1) == 1 || x.size(-1) == 1, "x must be contiguous along seqlen");
    const int64_t batch = x.size(0), dim = x.size(1), seqlen = x.size(2);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == dim, "weight must have shape (dim, width)");
    const int64_t width = weight.size(1);
    TORCH_CHECK(width >= 1 && width <= MM_CONV1D_MAX_WIDTH, "width must be between 1 and 8");
    at::Tensor out;
    if (out_.has_value()) {
        out = out_.value();
        CHECK_SHAPE(out, batch, dim, seqlen);
        TORCH_CHECK(out.is_cuda() && out.scalar_type() == x.scalar_type(), "out must have the dtype of x");
        TORCH_CHECK(out.stride(-1) == 1 || seqlen == 1, "out must be contiguous along seqlen");
    } else {
        out = torch::empty_like(x);
    }
    mm_conv1d_fwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.dim = dim; p.seqlen = seqlen; p.width = width;
    p.itype = conv_dtype(x, "x");
    p.wtype = conv_dtype(weight, "weight");
    p.silu = silu;
    p.x = x.data_ptr(); p.x_batch_stride = x.stride(0); p.x_d_stride = x.stride(1);
    p.out = out.data_ptr(); p.out_batch_stride = out.stride(0); p.out_d_stride = out.stride(1);
    p.weight = weight.data_ptr(); p.weight_d_stride = weight.stride(0); p.weight_w_stride = weight.stride(1);
    if (bias_.has_value()) {
        const at::Tensor &bias = bias_.value();
        TORCH_CHECK(bias.is_cuda() && bias.dim() == 1 && bias.size(0) == dim, "bias must have shape (dim,)");
        TORCH_CHECK(bias.scalar_type() == weight.scalar_type(), "bias must have the dtype of weight");
        p.bias = bias.data_ptr(); p.bias_stride = bias.stride(0);
    }
    if (initial_states_.has_value()) {
        const at::Tensor &ini = initial_states_.value();
        TORCH_CHECK(ini.is_cuda() && ini.dim() == 3 && ini.size(0) == batch && ini.size(1) == dim && ini.size(2) == width - 1,
                    "initial_states must have shape (batch, dim, width - 1)");
        TORCH_CHECK(ini.scalar_type() == x.scalar_type(), "initial_states must have the dtype of x");
        p.initial_states = ini.data_ptr();
        p.init_batch_stride = ini.stride(0); p.init_d_stride = ini.stride(1); p.init_w_stride = ini.stride(2);
    }
    if (final_states_out_.has_value()) {
        const at::Tensor &fin = final_states_out_.value();
        TORCH_CHECK(fin.is_cuda() && fin.dim() == 3 && fin.size(0) == batch && fin.size(1) == dim && fin.size(2) == width - 1,
                    "final_states_out must have shape (batch, dim, width - 1)");
        TORCH_CHECK(fin.scalar_type() == x.scalar_type(), "final_states_out must have the dtype of x");
        p.final_states = fin.data_ptr();
        p.final_batch_stride = fin.stride(0); p.final_d_stride = fin.stride(1); p.final_w_stride = fin.stride(2);
    }
    const c10::DeviceGuard device_guard{x.device()};
    check_rc(mm_causal_conv1d_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_causal_conv1d_fwd");
    return out;
}

// causal_conv1d_bwd (package causal-conv1d, as MambaInnerFn.backward calls it,
// selective_scan_interface.py:635-637): [dx, dweight, dbias?] for the gradient dout of the forward's
// output; dx is written into dx_out when given (MambaInnerFn passes a slice of dxz). dweight and dbias
// are summed in float32 and returned in the dtypes of weight and bias.
std::vector<at::Tensor> conv1d_bwd(const at::Tensor &x, const at::Tensor &weight, const c10::optional<at::Tensor> &bias_,
                                   const at::Tensor &dout, const c10::optional<at::Tensor> &dx_out_, bool silu) {
    TORCH_CHECK(x.is_cuda() && weight.is_cuda() && dout.is_cuda(), "x, weight and dout must be on the GPU");
    TORCH_CHECK(x.dim() == 3, "x must have shape (batch, dim, seqlen)");
    TORCH_CHECK(x.stride(-1) == 1 || x.size(-1) == 1, "x must be contiguous along seqlen");
    const int64_t batch = x.size(0), dim = x.size(1), seqlen = x.size(2);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == dim, "weight must have shape (dim, width)");
    const int64_t width = weight.size(1);
    TORCH_CHECK(width >= 1 && width <= MM_CONV1D_MAX_WIDTH, "width must be between 1 and 8");
    CHECK_SHAPE(dout, batch, dim, seqlen);
    TORCH_CHECK(dout.scalar_type() == x.scalar_type(), "dout must have the dtype of x");
    TORCH_CHECK(dout.stride(-1) == 1 || seqlen == 1, "dout must be contiguous along seqlen");
    at::Tensor dx;
    if (dx_out_.has_value()) {
        dx = dx_out_.value();
        CHECK_SHAPE(dx, batch, dim, seqlen);
        TORCH_CHECK(dx.is_cuda() && dx.scalar_type() == x.scalar_type(), "dx must have the dtype of x");
        TORCH_CHECK(dx.stride(-1) == 1 || seqlen == 1, "dx must be contiguous along seqlen");
    } else {
        dx = torch::empty_like(x);
    }
    at::Tensor dweight = torch::empty({dim, width}, x.options().dtype(at::kFloat));
    at::Tensor dbias;
    mm_conv1d_bwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.dim = dim; p.seqlen = seqlen; p.width = width;
    p.itype = conv_dtype(x, "x");
    p.wtype = conv_dtype(weight, "weight");
    p.silu = silu;
    p.x = x.data_ptr(); p.x_batch_stride = x.stride(0); p.x_d_stride = x.stride(1);
    p.dout = dout.data_ptr(); p.dout_batch_stride = dout.stride(0); p.dout_d_stride = dout.stride(1);
    p.dx = dx.data_ptr(); p.dx_batch_stride = dx.stride(0); p.dx_d_stride = dx.stride(1);
    p.weight = weight.data_ptr(); p.weight_d_stride = weight.stride(0); p.weight_w_stride = weight.stride(1);
    p.dweight = dweight.data_ptr<float>();
    if (bias_.has_value()) {
        const at::Tensor &bias = bias_.value();
        TORCH_CHECK(bias.is_cuda() && bias.dim() == 1 && bias.size(0) == dim, "bias must have shape (dim,)");
        TORCH_CHECK(bias.scalar_type() == weight.scalar_type(), "bias must have the dtype of weight");
        p.bias = bias.data_ptr(); p.bias_stride = bias.stride(0);
        dbias = torch::empty({dim}, x.options().dtype(at::kFloat));
        p.dbias = dbias.data_ptr<float>();
    }
    const c10::DeviceGuard device_guard{x.device()};
    check_rc(mm_causal_conv1d_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_causal_conv1d_bwd");
    std::vector<at::Tensor> res{dx, dweight.to(weight.scalar_type())};
    if (dbias.defined()) res.push_back(dbias.to(bias_.value().scalar_type()));
    return res;
}

// causal_conv1d_update (package causal-conv1d; fallback mamba_simplemotif.py:353-358): x (batch, dim)
// or (batch, dim, seqlen), conv_state (batch, dim, state_len) updated in place.
at::Tensor conv1d_update(const at::Tensor &x, const at::Tensor &conv_state, const at::Tensor &weight,
                         const c10::optional<at::Tensor> &bias_, bool silu) {
    TORCH_CHECK(x.is_cuda() && conv_state.is_cuda() && weight.is_cuda(), "x, conv_state and weight must be on the GPU");
    TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "x must have shape (batch, dim) or (batch, dim, seqlen)");
    const at::Tensor x3 = x.dim() == 2 ? x.unsqueeze(-1) : x;
    const int64_t batch = x3.size(0), dim = x3.size(1), seqlen = x3.size(2);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == dim, "weight must have shape (dim, width)");
    const int64_t width = weight.size(1);
    TORCH_CHECK(width >= 1 && width <= MM_CONV1D_MAX_WIDTH, "width must be between 1 and 8");
    TORCH_CHECK(conv_state.dim() == 3 && conv_state.size(0) == batch && conv_state.size(1) == dim,
                "conv_state must have shape (batch, dim, state_len)");
    TORCH_CHECK(conv_state.size(2) >= width - 1, "conv_state must hold at least width - 1 steps");
    at::Tensor out = torch::empty_like(x3);
    mm_conv1d_update_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.dim = dim; p.seqlen = seqlen; p.width = width; p.state_len = conv_state.size(2);
    p.itype = conv_dtype(x, "x");
    p.wtype = conv_dtype(weight, "weight");
    p.stype = conv_dtype(conv_state, "conv_state");
    p.silu = silu;
    p.x = x3.data_ptr(); p.x_batch_stride = x3.stride(0); p.x_d_stride = x3.stride(1); p.x_l_stride = x3.stride(2);
    p.conv_state = conv_state.data_ptr();
    p.state_batch_stride = conv_state.stride(0); p.state_d_stride = conv_state.stride(1);
    p.state_l_stride = conv_state.stride(2);
    p.out = out.data_ptr(); p.out_batch_stride = out.stride(0); p.out_d_stride = out.stride(1);
    p.out_l_stride = out.stride(2);
    p.weight = weight.data_ptr(); p.weight_d_stride = weight.stride(0); p.weight_w_stride = weight.stride(1);
    if (bias_.has_value()) {
        const at::Tensor &bias = bias_.value();
        TORCH_CHECK(bias.is_cuda() && bias.dim() == 1 && bias.size(0) == dim, "bias must have shape (dim,)");
        TORCH_CHECK(bias.scalar_type() == weight.scalar_type(), "bias must have the dtype of weight");
        p.bias = bias.data_ptr(); p.bias_stride = bias.stride(0);
    }
    const c10::DeviceGuard device_guard{x.device()};
    check_rc(mm_causal_conv1d_update(&p, c10::hip::getCurrentHIPStream().stream()), "mm_causal_conv1d_update");
    return x.dim() == 2 ? out.squeeze(-1) : out;
}

// rms_norm_forward (selective_scan_interface.py:217-234) over dim 1 of a 3-D x (n0, cols, n2), in
// the layout the scan reads: out[i0, :, i2] = x[i0, :, i2] * weight / rms. out is a new tensor with
// x's shape and dtype (x's layout when x is dense), or the given `out` (which may be x itself).
at::Tensor rms_norm_fwd(const at::Tensor &x, const at::Tensor &weight, double eps,
                        const c10::optional<at::Tensor> &out_) {
    TORCH_CHECK(x.is_cuda() && weight.is_cuda(), "x and weight must be on the GPU");
    TORCH_CHECK(x.dim() == 3, "x must have shape (n0, cols, n2)");
    const int64_t n0 = x.size(0), cols = x.size(1), n2 = x.size(2);
    CHECK_SHAPE(weight, cols);
    at::Tensor out = out_.has_value() ? out_.value() : torch::empty_like(x);
    CHECK_SHAPE(out, n0, cols, n2);
    TORCH_CHECK(out.is_cuda() && out.scalar_type() == x.scalar_type(), "out must have the dtype of x");
    mm_rms_norm_params p;
    std::memset(&p, 0, sizeof(p));
    p.n0 = n0; p.cols = cols; p.n2 = n2;
    p.itype = conv_dtype(x, "x");
    p.wtype = conv_dtype(weight, "weight");
    p.eps = static_cast<float>(eps);
    p.x = x.data_ptr(); p.weight = weight.data_ptr(); p.out = out.data_ptr();
    p.x_stride0 = x.stride(0); p.x_stride_c = x.stride(1); p.x_stride2 = x.stride(2);
    p.out_stride0 = out.stride(0); p.out_stride_c = out.stride(1); p.out_stride2 = out.stride(2);
    p.weight_stride = weight.stride(0);
    const c10::DeviceGuard device_guard{x.device()};
    check_rc(mm_rms_norm_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_rms_norm_fwd");
    return out;
}

at::Tensor state_update(const at::Tensor &state, const at::Tensor &x, const at::Tensor &dt, const at::Tensor &A,
                        const at::Tensor &B, const at::Tensor &C, const c10::optional<at::Tensor> &D_,
                        const c10::optional<at::Tensor> &z_, const c10::optional<at::Tensor> &dt_bias_,
                        bool dt_softplus) {
    TORCH_CHECK(state.dim() == 3, "state must have shape (batch, dim, dstate)");
    auto float_type = [](at::ScalarType t) {
        return t == at::ScalarType::Float || t == at::ScalarType::Half || t == at::ScalarType::BFloat16;
    };
    TORCH_CHECK(float_type(state.scalar_type()), "state must be float32, float16 or bfloat16");
    const int64_t batch = state.size(0), dim = state.size(1), dstate = state.size(2);
    const auto itype = x.scalar_type();
    TORCH_CHECK(state.is_cuda() && x.is_cuda() && dt.is_cuda() && A.is_cuda() && B.is_cuda() && C.is_cuda());
    CHECK_SHAPE(x, batch, dim);
    CHECK_SHAPE(dt, batch, dim);
    CHECK_SHAPE(A, dim, dstate);
    TORCH_CHECK(dt.scalar_type() == itype, "dt must have the dtype of x");
    TORCH_CHECK(A.scalar_type() == at::ScalarType::Float, "A must be float32");
    TORCH_CHECK(B.dim() == 2 || B.dim() == 3, "B must be (batch, dstate) or (batch, n_groups, dstate)");
    TORCH_CHECK(C.dim() == B.dim(), "B and C must have the same rank");
    const int64_t n_groups = B.dim() == 3 ? B.size(1) : 1;
    if (B.dim() == 2) {
        CHECK_SHAPE(B, batch, dstate);
        CHECK_SHAPE(C, batch, dstate);
    } else {
        CHECK_SHAPE(B, batch, n_groups, dstate);
        CHECK_SHAPE(C, batch, n_groups, dstate);
    }
    TORCH_CHECK(B.scalar_type() == itype && C.scalar_type() == itype, "B and C must have the dtype of x");
    TORCH_CHECK(n_groups >= 1 && dim % n_groups == 0, "dim must be a multiple of n_groups");
    if (D_.has_value()) {
        CHECK_SHAPE(D_.value(), dim);
        TORCH_CHECK(float_type(D_.value().scalar_type()) && D_.value().is_cuda(),
                    "D must be float32, float16 or bfloat16 on the GPU");
    }
    if (dt_bias_.has_value()) {
        CHECK_SHAPE(dt_bias_.value(), dim);
        TORCH_CHECK(float_type(dt_bias_.value().scalar_type()) && dt_bias_.value().is_cuda(),
                    "dt_bias must be float32, float16 or bfloat16 on the GPU");
    }
    if (z_.has_value()) {
        CHECK_SHAPE(z_.value(), batch, dim);
        TORCH_CHECK(z_.value().scalar_type() == itype && z_.value().is_cuda(), "z must have the dtype of x");
    }
    at::Tensor out = torch::empty({batch, dim}, x.options());
    at::Tensor Dc = D_.has_value() ? D_.value().contiguous() : at::Tensor();
    at::Tensor bc = dt_bias_.has_value() ? dt_bias_.value().contiguous() : at::Tensor();

    mm_state_update_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch;
    p.dim = dim;
    p.dstate = dstate;
    p.n_groups = n_groups;
    p.itype = to_mm(itype);
    p.dt_softplus = dt_softplus;
    p.state = state.data_ptr();
    p.state_type = to_mm(state.scalar_type());
    p.x = x.data_ptr();
    p.dt = dt.data_ptr();
    p.A = A.data_ptr<float>();
    p.B = B.data_ptr();
    p.C = C.data_ptr();
    p.D = Dc.defined() ? Dc.data_ptr() : nullptr;
    p.D_type = Dc.defined() ? to_mm(Dc.scalar_type()) : MM_FLOAT32;
    p.z = z_.has_value() ? z_.value().data_ptr() : nullptr;
    p.dt_bias = bc.defined() ? bc.data_ptr() : nullptr;
    p.dt_bias_type = bc.defined() ? to_mm(bc.scalar_type()) : MM_FLOAT32;
    p.out = out.data_ptr();
    p.state_batch_stride = state.stride(0);
    p.state_d_stride = state.stride(1);
    p.state_dstate_stride = state.stride(2);
    p.x_batch_stride = x.stride(0);
    p.x_d_stride = x.stride(1);
    p.dt_batch_stride = dt.stride(0);
    p.dt_d_stride = dt.stride(1);
    if (z_.has_value()) {
        p.z_batch_stride = z_.value().stride(0);
        p.z_d_stride = z_.value().stride(1);
    }
    p.out_batch_stride = out.stride(0);
    p.out_d_stride = out.stride(1);
    p.A_d_stride = A.stride(0);
    p.A_dstate_stride = A.stride(1);
    if (B.dim() == 3) {
        p.B_batch_stride = B.stride(0);
        p.B_group_stride = B.stride(1);
        p.B_dstate_stride = B.stride(2);
        p.C_batch_stride = C.stride(0);
        p.C_group_stride = C.stride(1);
        p.C_dstate_stride = C.stride(2);
    } else {
        p.B_batch_stride = B.stride(0);
        p.B_dstate_stride = B.stride(1);
        p.C_batch_stride = C.stride(0);
        p.C_dstate_stride = C.stride(1);
    }
    const c10::DeviceGuard device_guard{state.device()};
    check_rc(mm_state_update(&p, c10::hip::getCurrentHIPStream().stream()), "mm_state_update");
    return out;
}

// ---- linear attention and group norm --------------------------------------------------------------

mm_dtype float_dtype(const at::Tensor &t, const char *name) {
    const auto st = t.scalar_type();
    TORCH_CHECK(st == at::ScalarType::Float || st == at::ScalarType::Half || st == at::ScalarType::BFloat16, name,
                " must be float32, float16 or bfloat16");
    return to_mm(st);
}

// q, k (lead..., groups, dk) and v (lead..., heads, dv), on one device and of one dtype, rows contiguous.
void check_qkv(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, int64_t rank) {
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "q, k and v must be on the GPU");
    TORCH_CHECK(q.device() == v.device() && k.device() == v.device(), "q, k and v must be on one device");
    TORCH_CHECK(q.dim() == rank && v.dim() == rank, "q, k and v must have ", rank, " dimensions");
    TORCH_CHECK(q.sizes() == k.sizes(), "q and k must have the same shape");
    for (int64_t i = 0; i < rank - 2; ++i) TORCH_CHECK(q.size(i) == v.size(i), "q, k and v must agree in batch and seqlen");
    TORCH_CHECK(q.scalar_type() == v.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
    float_dtype(v, "v");
    for (const auto *t : {&q, &k, &v}) TORCH_CHECK(t->stride(-1) == 1 || t->size(-1) == 1, "q, k and v must be contiguous along their last dimension");
    const int64_t groups = q.size(-2), heads = v.size(-2);
    TORCH_CHECK(groups >= 1 && heads % groups == 0, "the heads of v must be a multiple of those of q and k");
    TORCH_CHECK(q.size(-1) >= 1 && v.size(-1) >= 1, "q, k and v must have at least one element per head");
}

void check_decay(const at::Tensor &g, at::IntArrayRef sizes, const at::Tensor &v) {
    TORCH_CHECK(g.is_cuda() && g.device() == v.device(), "log_decay must be on the device of v");
    TORCH_CHECK(g.sizes() == sizes, "log_decay must have the shape of v without its last dimension, or (nheads,)");
    float_dtype(g, "log_decay");
}

void check_state(const at::Tensor &s, const at::Tensor &v, int64_t batch, int64_t heads, int64_t dk, int64_t dv, const char *name) {
    TORCH_CHECK(s.is_cuda() && s.device() == v.device(), name, " must be on the device of v");
    TORCH_CHECK(s.scalar_type() == at::ScalarType::Float, name, " must be float32");
    TORCH_CHECK(s.sizes() == torch::IntArrayRef({batch, heads, dk, dv}), name, " must have shape (batch, nheads, dk, dv)");
}

// The stride between tokens; a single token has none, whatever its tensor says.
int64_t seq_stride(const at::Tensor &t) { return t.size(1) > 1 ? t.stride(1) : 0; }

void *workspace_of(at::Tensor &keep, int64_t bytes, const at::Tensor &like) {
    if (bytes <= 0) return nullptr;
    keep = torch::empty({bytes}, like.options().dtype(at::ScalarType::Byte));
    return keep.data_ptr();
}

std::vector<at::Tensor> linattn_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                                    double scale, const c10::optional<at::Tensor> &initial_, bool return_last_state, bool keep_states) {
    check_qkv(q, k, v, 4);
    const int64_t batch = v.size(0), seqlen = v.size(1), heads = v.size(2), dv = v.size(3), dk = q.size(3);
    check_decay(g, {batch, seqlen, heads}, v);
    at::Tensor initial;
    if (initial_.has_value()) {
        check_state(initial_.value(), v, batch, heads, dk, dv, "initial_state");
        initial = initial_.value().contiguous();
    }
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor out = torch::empty({batch, seqlen, heads, dv}, v.options());
    at::Tensor last;
    if (return_last_state) last = torch::empty({batch, heads, dk, dv}, v.options().dtype(at::ScalarType::Float));
    mm_linattn_fwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.seqlen = seqlen; p.n_groups = q.size(2); p.nheads = heads; p.dk = dk; p.dv = dv;
    p.itype = to_mm(v.scalar_type());
    p.gtype = to_mm(g.scalar_type());
    p.scale = static_cast<float>(scale);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.log_decay = g.data_ptr();
    p.initial_state = initial.defined() ? initial.data_ptr<float>() : nullptr;
    p.out = out.data_ptr();
    p.last_state = last.defined() ? last.data_ptr<float>() : nullptr;
    p.q_batch_stride = q.stride(0); p.q_seq_stride = seq_stride(q); p.q_group_stride = q.stride(2);
    p.k_batch_stride = k.stride(0); p.k_seq_stride = seq_stride(k); p.k_group_stride = k.stride(2);
    p.v_batch_stride = v.stride(0); p.v_seq_stride = seq_stride(v); p.v_head_stride = v.stride(2);
    p.g_batch_stride = g.stride(0); p.g_seq_stride = g.stride(1); p.g_head_stride = g.stride(2);
    p.out_batch_stride = out.stride(0); p.out_seq_stride = seq_stride(out); p.out_head_stride = out.stride(2);
    at::Tensor ws;
    p.workspace_bytes = mm_linattn_fwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, v);
    check_rc(mm_linattn_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_linattn_fwd");
    std::vector<at::Tensor> res{out};
    if (return_last_state) res.push_back(last);
    if (keep_states) res.push_back(ws);   // undefined where a row is one segment
    return res;
}

// Gradients [dq, dk, dv, dlog_decay | None, dinitial_state | None]; dlog_decay has the shape of log_decay, or
// (nheads,) with decay_per_head.
std::vector<c10::optional<at::Tensor>> linattn_bwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                                                   double scale, const c10::optional<at::Tensor> &initial_, const at::Tensor &dout,
                                                   const c10::optional<at::Tensor> &dlast_, const c10::optional<at::Tensor> &states_,
                                                   bool decay_per_head, bool want_decay, bool want_initial) {
    check_qkv(q, k, v, 4);
    const int64_t batch = v.size(0), seqlen = v.size(1), heads = v.size(2), dv = v.size(3), dk = q.size(3);
    check_decay(g, {batch, seqlen, heads}, v);
    TORCH_CHECK(dout.is_cuda() && dout.sizes() == v.sizes() && dout.scalar_type() == v.scalar_type(), "dout must have the shape and dtype of v");
    TORCH_CHECK(dout.stride(-1) == 1 || dout.size(-1) == 1, "dout must be contiguous along its last dimension");
    at::Tensor initial, dlast;
    if (initial_.has_value()) {
        check_state(initial_.value(), v, batch, heads, dk, dv, "initial_state");
        initial = initial_.value().contiguous();
    }
    if (dlast_.has_value()) {
        check_state(dlast_.value(), v, batch, heads, dk, dv, "dlast_state");
        dlast = dlast_.value().contiguous();
    }
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor dq = torch::empty(q.sizes(), q.options()), dkk = torch::empty(k.sizes(), k.options()), dvv = torch::empty(v.sizes(), v.options());
    at::Tensor dg, ds;
    if (want_decay) dg = decay_per_head ? torch::empty({heads}, g.options()) : torch::empty({batch, seqlen, heads}, g.options());
    if (want_initial) ds = torch::empty({batch, heads, dk, dv}, v.options().dtype(at::ScalarType::Float));
    mm_linattn_bwd_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.seqlen = seqlen; p.n_groups = q.size(2); p.nheads = heads; p.dk = dk; p.dv = dv;
    p.itype = to_mm(v.scalar_type());
    p.gtype = to_mm(g.scalar_type());
    p.scale = static_cast<float>(scale);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.log_decay = g.data_ptr();
    p.initial_state = initial.defined() ? initial.data_ptr<float>() : nullptr;
    p.dout = dout.data_ptr();
    p.dlast_state = dlast.defined() ? dlast.data_ptr<float>() : nullptr;
    p.dq = dq.data_ptr(); p.dk_out = dkk.data_ptr(); p.dv_out = dvv.data_ptr();
    p.dlog_decay = dg.defined() ? dg.data_ptr() : nullptr;
    p.dinitial_state = ds.defined() ? ds.data_ptr<float>() : nullptr;
    p.decay_per_head = decay_per_head;
    p.segment_states = states_.has_value() && states_.value().defined() ? states_.value().data_ptr() : nullptr;
    p.q_batch_stride = q.stride(0); p.q_seq_stride = seq_stride(q); p.q_group_stride = q.stride(2);
    p.k_batch_stride = k.stride(0); p.k_seq_stride = seq_stride(k); p.k_group_stride = k.stride(2);
    p.v_batch_stride = v.stride(0); p.v_seq_stride = seq_stride(v); p.v_head_stride = v.stride(2);
    p.g_batch_stride = g.stride(0); p.g_seq_stride = g.stride(1); p.g_head_stride = g.stride(2);
    p.do_batch_stride = dout.stride(0); p.do_seq_stride = seq_stride(dout); p.do_head_stride = dout.stride(2);
    at::Tensor ws;
    p.workspace_bytes = mm_linattn_bwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, v);
    check_rc(mm_linattn_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_linattn_bwd");
    std::vector<c10::optional<at::Tensor>> res{dq, dkk, dvv, c10::nullopt, c10::nullopt};
    if (want_decay) res[3] = dg;
    if (want_initial) res[4] = ds;
    return res;
}

at::Tensor linattn_update(const at::Tensor &state, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                          double scale) {
    check_qkv(q, k, v, 3);
    const int64_t batch = v.size(0), heads = v.size(1), dv = v.size(2), dk = q.size(2);
    check_decay(g, {batch, heads}, v);
    check_state(state, v, batch, heads, dk, dv, "state");
    TORCH_CHECK(state.stride(-1) == 1 || dv == 1, "state must be contiguous along its last dimension");
    for (const auto *t : {&state, &q, &k, &v, &g})
        TORCH_CHECK(!(at::GradMode::is_enabled() && t->requires_grad()) && !t->_fw_grad(0).defined(),
                    "linear_attention_update has no derivatives: call it under torch.no_grad() or on detached tensors");
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor out = torch::empty({batch, heads, dv}, v.options());
    mm_linattn_update_params p;
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.n_groups = q.size(1); p.nheads = heads; p.dk = dk; p.dv = dv;
    p.itype = to_mm(v.scalar_type());
    p.gtype = to_mm(g.scalar_type());
    p.scale = static_cast<float>(scale);
    p.state = state.data_ptr<float>();
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.log_decay = g.data_ptr();
    p.out = out.data_ptr();
    p.state_batch_stride = state.stride(0); p.state_head_stride = state.stride(1); p.state_dk_stride = state.stride(2);
    p.q_batch_stride = q.stride(0); p.q_group_stride = q.stride(1);
    p.k_batch_stride = k.stride(0); p.k_group_stride = k.stride(1);
    p.v_batch_stride = v.stride(0); p.v_head_stride = v.stride(1);
    p.g_batch_stride = g.stride(0); p.g_head_stride = g.stride(1);
    check_rc(mm_linattn_update(&p, c10::hip::getCurrentHIPStream().stream()), "mm_linattn_update");
    // The state is not what an autograd node may have saved any more.
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return out;
}

mm_group_norm_params norm_params(const at::Tensor &x, int64_t n_groups, const c10::optional<at::Tensor> &weight_,
                                 const c10::optional<at::Tensor> &bias_, const c10::optional<at::Tensor> &z_, double eps, bool is_rms,
                                 int64_t gate) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a (rows, channels) tensor on the GPU");
    const int64_t rows = x.size(0), channels = x.size(1);
    auto row_ok = [&](const at::Tensor &t) { return t.stride(1) == 1 || channels == 1; };
    TORCH_CHECK(row_ok(x), "x must be contiguous along its channels");
    TORCH_CHECK(n_groups >= 1 && channels % n_groups == 0, "the channels must be a multiple of n_groups");
    mm_group_norm_params p;
    std::memset(&p, 0, sizeof(p));
    p.rows = rows; p.channels = channels; p.n_groups = n_groups;
    p.itype = float_dtype(x, "x");
    p.wtype = MM_FLOAT32;
    p.eps = static_cast<float>(eps);
    p.is_rms = is_rms;
    p.gate = static_cast<mm_gate>(gate);
    p.x = x.data_ptr();
    p.x_row_stride = x.stride(0);
    for (const auto *t : {&weight_, &bias_})
        if (t->has_value()) {
            const at::Tensor &w = t->value();
            TORCH_CHECK(w.is_cuda() && w.device() == x.device() && w.dim() == 1 && w.size(0) == channels && w.is_contiguous(),
                        "weight and bias must be contiguous (channels,) tensors on the device of x");
            p.wtype = float_dtype(w, "weight");
        }
    if (weight_.has_value() && bias_.has_value())
        TORCH_CHECK(weight_.value().scalar_type() == bias_.value().scalar_type(), "weight and bias must have one dtype");
    p.weight = weight_.has_value() ? weight_.value().data_ptr() : nullptr;
    p.bias = bias_.has_value() ? bias_.value().data_ptr() : nullptr;
    if (z_.has_value()) {
        const at::Tensor &z = z_.value();
        TORCH_CHECK(z.is_cuda() && z.device() == x.device() && z.sizes() == x.sizes() && z.scalar_type() == x.scalar_type(),
                    "z must have the shape, dtype and device of x");
        TORCH_CHECK(row_ok(z), "z must be contiguous along its channels");
        p.z = z.data_ptr();
        p.z_row_stride = z.stride(0);
    }
    return p;
}

at::Tensor group_norm_fwd(const at::Tensor &x, int64_t n_groups, const c10::optional<at::Tensor> &weight, const c10::optional<at::Tensor> &bias,
                          const c10::optional<at::Tensor> &z, double eps, bool is_rms, int64_t gate) {
    mm_group_norm_params p = norm_params(x, n_groups, weight, bias, z, eps, is_rms, gate);
    const c10::DeviceGuard device_guard{x.device()};
    at::Tensor out = torch::empty({p.rows, p.channels}, x.options());
    p.out = out.data_ptr();
    check_rc(mm_group_norm_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_group_norm_fwd");
    return out;
}

// [dx, dweight | None, dbias | None, dz | None]
std::vector<c10::optional<at::Tensor>> group_norm_bwd(const at::Tensor &x, int64_t n_groups, const c10::optional<at::Tensor> &weight,
                                                      const c10::optional<at::Tensor> &bias, const c10::optional<at::Tensor> &z, double eps,
                                                      bool is_rms, int64_t gate, const at::Tensor &dout, bool want_weights) {
    mm_group_norm_params p = norm_params(x, n_groups, weight, bias, z, eps, is_rms, gate);
    TORCH_CHECK(dout.is_cuda() && dout.sizes() == x.sizes() && dout.scalar_type() == x.scalar_type(), "dout must have the shape and dtype of x");
    TORCH_CHECK(dout.stride(1) == 1 || p.channels == 1, "dout must be contiguous along its channels");
    const c10::DeviceGuard device_guard{x.device()};
    std::vector<c10::optional<at::Tensor>> res{torch::empty({p.rows, p.channels}, x.options()), c10::nullopt, c10::nullopt, c10::nullopt};
    p.dout = dout.data_ptr();
    p.dout_row_stride = dout.stride(0);
    p.dx = res[0].value().data_ptr();
    if (want_weights && weight.has_value()) {
        res[1] = torch::empty_like(weight.value());
        p.dweight = res[1].value().data_ptr();
    }
    if (want_weights && bias.has_value()) {
        res[2] = torch::empty_like(bias.value());
        p.dbias = res[2].value().data_ptr();
    }
    if (z.has_value()) {
        res[3] = torch::empty({p.rows, p.channels}, x.options());
        p.dz = res[3].value().data_ptr();
    }
    at::Tensor ws;
    p.workspace_bytes = mm_group_norm_bwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, x);
    check_rc(mm_group_norm_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_group_norm_bwd");
    return res;
}

// ---- gated delta rule ----------------------------------------------------------------------------

void check_beta(const at::Tensor &b, at::IntArrayRef sizes, const at::Tensor &v) {
    TORCH_CHECK(b.is_cuda() && b.device() == v.device(), "beta must be on the device of v");
    TORCH_CHECK(b.sizes() == sizes, "beta must have the shape of v without its last dimension");
    float_dtype(b, "beta");
}

// The fields that the forward and backward have alike.
template <typename P>
void delta_common(P &p, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &b, const c10::optional<at::Tensor> &g_, double scale) {
    check_qkv(q, k, v, 4);
    const int64_t batch = v.size(0), seqlen = v.size(1), heads = v.size(2);
    check_beta(b, {batch, seqlen, heads}, v);
    std::memset(&p, 0, sizeof(p));
    p.batch = batch; p.seqlen = seqlen; p.n_groups = q.size(2); p.nheads = heads; p.dk = q.size(3); p.dv = v.size(3);
    p.itype = to_mm(v.scalar_type());
    p.btype = to_mm(b.scalar_type());
    p.gtype = MM_FLOAT32;
    p.scale = static_cast<float>(scale);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.beta = b.data_ptr();
    p.q_batch_stride = q.stride(0); p.q_seq_stride = seq_stride(q); p.q_group_stride = q.stride(2);
    p.k_batch_stride = k.stride(0); p.k_seq_stride = seq_stride(k); p.k_group_stride = k.stride(2);
    p.v_batch_stride = v.stride(0); p.v_seq_stride = seq_stride(v); p.v_head_stride = v.stride(2);
    p.b_batch_stride = b.stride(0); p.b_seq_stride = b.stride(1); p.b_head_stride = b.stride(2);
    if (g_.has_value()) {
        const at::Tensor &g = g_.value();
        check_decay(g, {batch, seqlen, heads}, v);
        p.gtype = to_mm(g.scalar_type());
        p.log_decay = g.data_ptr();
        p.g_batch_stride = g.stride(0); p.g_seq_stride = g.stride(1); p.g_head_stride = g.stride(2);
    }
}

std::vector<at::Tensor> delta_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &b, const c10::optional<at::Tensor> &g,
                                  double scale, const c10::optional<at::Tensor> &initial_, bool return_last_state, bool keep_states) {
    mm_delta_fwd_params p;
    delta_common(p, q, k, v, b, g, scale);
    at::Tensor initial;
    if (initial_.has_value()) {
        check_state(initial_.value(), v, p.batch, p.nheads, p.dk, p.dv, "initial_state");
        initial = initial_.value().contiguous();
    }
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor out = torch::empty({p.batch, p.seqlen, p.nheads, p.dv}, v.options());
    at::Tensor last;
    if (return_last_state) last = torch::empty({p.batch, p.nheads, p.dk, p.dv}, v.options().dtype(at::ScalarType::Float));
    p.initial_state = initial.defined() ? initial.data_ptr<float>() : nullptr;
    p.out = out.data_ptr();
    p.last_state = last.defined() ? last.data_ptr<float>() : nullptr;
    p.out_batch_stride = out.stride(0); p.out_seq_stride = seq_stride(out); p.out_head_stride = out.stride(2);
    at::Tensor ws, kept;
    if (keep_states) {
        p.segment_states_bytes = mm_delta_segment_states_size(&p);
        p.segment_states = workspace_of(kept, p.segment_states_bytes, v);
    }
    p.workspace_bytes = mm_delta_fwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, v);
    check_rc(mm_delta_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_delta_fwd");
    std::vector<at::Tensor> res{out};
    if (return_last_state) res.push_back(last);
    if (keep_states) res.push_back(kept);   // undefined where a row is one segment
    return res;
}

// Gradients [dq, dk, dv, dbeta, dlog_decay | None, dinitial_state | None]; dlog_decay has the shape of log_decay, or (nheads,) with
// decay_per_head.
std::vector<c10::optional<at::Tensor>> delta_bwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &b,
                                                 const c10::optional<at::Tensor> &g, double scale, const c10::optional<at::Tensor> &initial_,
                                                 const at::Tensor &dout, const c10::optional<at::Tensor> &dlast_, const c10::optional<at::Tensor> &states_,
                                                 bool decay_per_head, bool want_decay, bool want_initial) {
    mm_delta_bwd_params p;
    delta_common(p, q, k, v, b, g, scale);
    TORCH_CHECK(dout.is_cuda() && dout.sizes() == v.sizes() && dout.scalar_type() == v.scalar_type(), "dout must have the shape and dtype of v");
    TORCH_CHECK(dout.stride(-1) == 1 || dout.size(-1) == 1 || dout.numel() == 0, "dout must be contiguous along its last dimension");
    at::Tensor initial, dlast;
    if (initial_.has_value()) {
        check_state(initial_.value(), v, p.batch, p.nheads, p.dk, p.dv, "initial_state");
        initial = initial_.value().contiguous();
    }
    if (dlast_.has_value()) {
        check_state(dlast_.value(), v, p.batch, p.nheads, p.dk, p.dv, "dlast_state");
        dlast = dlast_.value().contiguous();
    }
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor dq = torch::empty(q.sizes(), q.options()), dkk = torch::empty(k.sizes(), k.options()), dvv = torch::empty(v.sizes(), v.options());
    at::Tensor db = torch::empty(b.sizes(), b.options()), dg, ds;
    if (want_decay && g.has_value())
        dg = decay_per_head ? torch::empty({p.nheads}, g.value().options()) : torch::empty({p.batch, p.seqlen, p.nheads}, g.value().options());
    if (want_initial) ds = torch::empty({p.batch, p.nheads, p.dk, p.dv}, v.options().dtype(at::ScalarType::Float));
    p.initial_state = initial.defined() ? initial.data_ptr<float>() : nullptr;
    p.dout = dout.data_ptr();
    p.dlast_state = dlast.defined() ? dlast.data_ptr<float>() : nullptr;
    p.dq = dq.data_ptr(); p.dk_out = dkk.data_ptr(); p.dv_out = dvv.data_ptr(); p.dbeta = db.data_ptr();
    p.dlog_decay = dg.defined() ? dg.data_ptr() : nullptr;
    p.dinitial_state = ds.defined() ? ds.data_ptr<float>() : nullptr;
    p.decay_per_head = decay_per_head;
    if (states_.has_value() && states_.value().defined()) {
        p.segment_states = states_.value().data_ptr();
        p.segment_states_bytes = int64_t(states_.value().nbytes());
    }
    p.do_batch_stride = dout.stride(0); p.do_seq_stride = seq_stride(dout); p.do_head_stride = dout.stride(2);
    at::Tensor ws;
    p.workspace_bytes = mm_delta_bwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, v);
    check_rc(mm_delta_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_delta_bwd");
    std::vector<c10::optional<at::Tensor>> res{dq, dkk, dvv, db, c10::nullopt, c10::nullopt};
    if (dg.defined()) res[4] = dg;
    if (want_initial) res[5] = ds;
    return res;
}

at::Tensor delta_update(const at::Tensor &state, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &b,
                        const c10::optional<at::Tensor> &g_, double scale) {
    check_qkv(q, k, v, 3);
    const int64_t batch = v.size(0), heads = v.size(1), dv = v.size(2), dk = q.size(2);
    check_beta(b, {batch, heads}, v);
    check_state(state, v, batch, heads, dk, dv, "state");
    TORCH_CHECK(state.stride(-1) == 1 || dv == 1, "state must be contiguous along its last dimension");
    auto no_derivative = [](const at::Tensor &t) {
        TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()) && !t._fw_grad(0).defined(),
                    "delta_rule_update has no derivatives: call it under torch.no_grad() or on detached tensors");
    };
    for (const auto *t : {&state, &q, &k, &v, &b}) no_derivative(*t);
    mm_delta_update_params p;
    std::memset(&p, 0, sizeof(p));
    p.gtype = MM_FLOAT32;
    if (g_.has_value()) {
        const at::Tensor &g = g_.value();
        check_decay(g, {batch, heads}, v);
        no_derivative(g);
        p.gtype = to_mm(g.scalar_type());
        p.log_decay = g.data_ptr();
        p.g_batch_stride = g.stride(0); p.g_head_stride = g.stride(1);
    }
    const c10::DeviceGuard device_guard{v.device()};
    at::Tensor out = torch::empty({batch, heads, dv}, v.options());
    p.batch = batch; p.n_groups = q.size(1); p.nheads = heads; p.dk = dk; p.dv = dv;
    p.itype = to_mm(v.scalar_type());
    p.btype = to_mm(b.scalar_type());
    p.scale = static_cast<float>(scale);
    p.state = state.data_ptr<float>();
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.beta = b.data_ptr();
    p.out = out.data_ptr();
    p.state_batch_stride = state.stride(0); p.state_head_stride = state.stride(1); p.state_dk_stride = state.stride(2);
    p.q_batch_stride = q.stride(0); p.q_group_stride = q.stride(1);
    p.k_batch_stride = k.stride(0); p.k_group_stride = k.stride(1);
    p.v_batch_stride = v.stride(0); p.v_head_stride = v.stride(1);
    p.b_batch_stride = b.stride(0); p.b_head_stride = b.stride(1);
    check_rc(mm_delta_update(&p, c10::hip::getCurrentHIPStream().stream()), "mm_delta_update");
    // The state is not what an autograd node may have saved any more.
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return out;
}

// ---- layer norm ----------------------------------------------------------------------------------

// x or residual (rows, channels); x None: residual is h already.
mm_layer_norm_params layer_norm_params(const c10::optional<at::Tensor> &x_, const c10::optional<at::Tensor> &residual_, at::ScalarType rtype,
                                       const c10::optional<at::Tensor> &weight_, const c10::optional<at::Tensor> &bias_, double eps, bool is_rms,
                                       at::ScalarType itype) {
    const at::Tensor &ref = x_.has_value() ? x_.value() : residual_.value();
    TORCH_CHECK(ref.is_cuda() && ref.dim() == 2, "x must be a (rows, channels) tensor on the GPU");
    const int64_t rows = ref.size(0), channels = ref.size(1);
    TORCH_CHECK(itype == at::ScalarType::Float || itype == at::ScalarType::Half || itype == at::ScalarType::BFloat16, "x must be float32, float16 or bfloat16");
    mm_layer_norm_params p;
    std::memset(&p, 0, sizeof(p));
    p.rows = rows; p.channels = channels;
    p.itype = to_mm(itype);
    TORCH_CHECK(rtype == itype || rtype == at::ScalarType::Float, "residual must have x's dtype or float32");
    p.rtype = to_mm(rtype);
    p.wtype = MM_FLOAT32;
    p.eps = static_cast<float>(eps);
    p.is_rms = is_rms;
    for (const auto *t : {&x_, &residual_})
        if (t->has_value()) {
            const at::Tensor &r = t->value();
            TORCH_CHECK(r.is_cuda() && r.device() == ref.device() && r.sizes() == ref.sizes(), "residual must have the shape and device of x");
            TORCH_CHECK(r.scalar_type() == (t == &x_ ? itype : rtype), "residual has another dtype than stated");
            TORCH_CHECK(r.stride(1) == 1 || channels == 1 || rows == 0, "x and residual must be contiguous along their channels");
        }
    if (x_.has_value()) {
        p.x = x_.value().data_ptr();
        p.x_row_stride = x_.value().stride(0);
    }
    if (residual_.has_value()) {
        p.residual = residual_.value().data_ptr();
        p.residual_row_stride = residual_.value().stride(0);
    }
    for (const auto *t : {&weight_, &bias_})
        if (t->has_value()) {
            const at::Tensor &w = t->value();
            TORCH_CHECK(w.is_cuda() && w.device() == ref.device() && w.dim() == 1 && w.size(0) == channels && w.is_contiguous(),
                        "weight and bias must be contiguous (channels,) tensors on the device of x");
            p.wtype = float_dtype(w, "weight");
        }
    if (weight_.has_value() && bias_.has_value())
        TORCH_CHECK(weight_.value().scalar_type() == bias_.value().scalar_type(), "weight and bias must have one dtype");
    p.weight = weight_.has_value() ? weight_.value().data_ptr() : nullptr;
    p.bias = bias_.has_value() ? bias_.value().data_ptr() : nullptr;
    return p;
}

// [out, residual_out | None]; wide: residual_out in float32 where there is no residual that gives its dtype.
std::vector<c10::optional<at::Tensor>> layer_norm_fwd(const at::Tensor &x, const c10::optional<at::Tensor> &residual, const c10::optional<at::Tensor> &weight,
                                                      const c10::optional<at::Tensor> &bias, double eps, bool is_rms, bool want_residual, bool wide) {
    const at::ScalarType rtype = residual.has_value() ? residual.value().scalar_type() : wide ? at::ScalarType::Float : x.scalar_type();
    mm_layer_norm_params p = layer_norm_params(x, residual, rtype, weight, bias, eps, is_rms, x.scalar_type());
    const c10::DeviceGuard device_guard{x.device()};
    std::vector<c10::optional<at::Tensor>> res{torch::empty({p.rows, p.channels}, x.options()), c10::nullopt};
    p.out = res[0].value().data_ptr();
    if (want_residual) {
        res[1] = torch::empty({p.rows, p.channels}, x.options().dtype(rtype));
        p.residual_out = res[1].value().data_ptr();
    }
    check_rc(mm_layer_norm_fwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_layer_norm_fwd");
    return res;
}

// [dx | None, dresidual | None, dweight | None, dbias | None]
std::vector<c10::optional<at::Tensor>> layer_norm_bwd(const c10::optional<at::Tensor> &x, const c10::optional<at::Tensor> &residual,
                                                      const c10::optional<at::Tensor> &weight, const c10::optional<at::Tensor> &bias, double eps, bool is_rms,
                                                      const at::Tensor &dout, const c10::optional<at::Tensor> &dres, bool wide, bool want_dx, bool want_dres,
                                                      bool want_weight, bool want_bias) {
    const at::ScalarType rtype = wide ? at::ScalarType::Float : dout.scalar_type();
    mm_layer_norm_params p = layer_norm_params(x, residual, rtype, weight, bias, eps, is_rms, dout.scalar_type());
    const at::Tensor &ref = x.has_value() ? x.value() : residual.value();
    TORCH_CHECK(dout.is_cuda() && dout.device() == ref.device() && dout.sizes() == ref.sizes(), "dout must have the shape and device of x");
    TORCH_CHECK(dout.stride(1) == 1 || p.channels == 1 || p.rows == 0, "dout must be contiguous along its channels");
    p.dout = dout.data_ptr();
    p.dout_row_stride = dout.stride(0);
    if (dres.has_value()) {
        const at::Tensor &d = dres.value();
        TORCH_CHECK(d.is_cuda() && d.device() == ref.device() && d.sizes() == ref.sizes() && d.scalar_type() == rtype, "dresidual_out must have the shape, dtype and device of residual_out");
        TORCH_CHECK(d.stride(1) == 1 || p.channels == 1 || p.rows == 0, "dresidual_out must be contiguous along its channels");
        p.dresidual_out = d.data_ptr();
        p.dresidual_out_row_stride = d.stride(0);
    }
    const c10::DeviceGuard device_guard{ref.device()};
    std::vector<c10::optional<at::Tensor>> res{c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt};
    if (want_dx) {
        res[0] = torch::empty({p.rows, p.channels}, dout.options());
        p.dx = res[0].value().data_ptr();
    }
    if (want_dres) {
        res[1] = torch::empty({p.rows, p.channels}, dout.options().dtype(rtype));
        p.dresidual = res[1].value().data_ptr();
    }
    if (want_weight && weight.has_value()) {
        res[2] = torch::empty_like(weight.value());
        p.dweight = res[2].value().data_ptr();
    }
    if (want_bias && bias.has_value()) {
        res[3] = torch::empty_like(bias.value());
        p.dbias = res[3].value().data_ptr();
    }
    at::Tensor ws;
    p.workspace_bytes = mm_layer_norm_bwd_workspace_size(&p);
    p.workspace = workspace_of(ws, p.workspace_bytes, dout);
    check_rc(mm_layer_norm_bwd(&p, c10::hip::getCurrentHIPStream().stream()), "mm_layer_norm_bwd");
    return res;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("fwd", &fwd, "Selective scan forward (reference-compatible outputs [out, x, out_z?])",
          pybind11::arg("u"), pybind11::arg("delta"), pybind11::arg("A"), pybind11::arg("B"), pybind11::arg("C"),
          pybind11::arg("D") = pybind11::none(), pybind11::arg("z") = pybind11::none(),
          pybind11::arg("delta_bias") = pybind11::none(), pybind11::arg("P") = pybind11::none(),
          pybind11::arg("Q") = pybind11::none(), pybind11::arg("gamma") = pybind11::none(),
          pybind11::arg("delta_softplus") = false, pybind11::arg("tile_states") = false);
    m.def("bwd", &bwd, "Selective scan backward (reference-compatible outputs)",
          pybind11::arg("u"), pybind11::arg("delta"), pybind11::arg("A"), pybind11::arg("B"), pybind11::arg("C"),
          pybind11::arg("D") = pybind11::none(), pybind11::arg("z") = pybind11::none(),
          pybind11::arg("delta_bias") = pybind11::none(), pybind11::arg("P") = pybind11::none(),
          pybind11::arg("Q") = pybind11::none(), pybind11::arg("gamma") = pybind11::none(), pybind11::arg("dout"),
          pybind11::arg("x"), pybind11::arg("out"), pybind11::arg("dz"), pybind11::arg("dP_out") = pybind11::none(),
          pybind11::arg("dQ_out") = pybind11::none(), pybind11::arg("delta_softplus"),
          pybind11::arg("recompute_out_z"), pybind11::arg("tile_states") = pybind11::none());
    m.def("fwd_infer", &fwd_infer, "Selective scan forward, inference outputs [out_z|out, last_state?]",
          pybind11::arg("u"), pybind11::arg("delta"), pybind11::arg("A"), pybind11::arg("B"), pybind11::arg("C"),
          pybind11::arg("D") = pybind11::none(), pybind11::arg("z") = pybind11::none(),
          pybind11::arg("delta_bias") = pybind11::none(), pybind11::arg("delta_softplus") = false,
          pybind11::arg("return_last_state") = false, pybind11::arg("P") = pybind11::none(),
          pybind11::arg("Q") = pybind11::none(), pybind11::arg("gamma") = pybind11::none());
    m.def("state_update", &state_update, "Single-token selective state update (in place on state)",
          pybind11::arg("state"), pybind11::arg("x"), pybind11::arg("dt"), pybind11::arg("A"), pybind11::arg("B"),
          pybind11::arg("C"), pybind11::arg("D") = pybind11::none(), pybind11::arg("z") = pybind11::none(),
          pybind11::arg("dt_bias") = pybind11::none(), pybind11::arg("dt_softplus") = false);
    m.def("conv1d_fwd", &conv1d_fwd, "Causal depthwise conv1d forward",
          pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("bias") = pybind11::none(),
          pybind11::arg("initial_states") = pybind11::none(), pybind11::arg("final_states_out") = pybind11::none(),
          pybind11::arg("silu") = false, pybind11::arg("out") = pybind11::none());
    m.def("conv1d_bwd", &conv1d_bwd, "Causal depthwise conv1d backward [dx, dweight, dbias?]",
          pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("dout"),
          pybind11::arg("dx") = pybind11::none(), pybind11::arg("silu") = false);
    m.def("conv1d_update", &conv1d_update, "Causal depthwise conv1d decode update (in place on conv_state)",
          pybind11::arg("x"), pybind11::arg("conv_state"), pybind11::arg("weight"),
          pybind11::arg("bias") = pybind11::none(), pybind11::arg("silu") = false);
    m.def("rms_norm_fwd", &rms_norm_fwd, "Row RMSNorm over dim 1 of a 3-D tensor",
          pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("eps") = 1e-6,
          pybind11::arg("out") = pybind11::none());
    m.def("linattn_fwd", &linattn_fwd, "Linear attention forward [out, last_state?, states of the segments?]", pybind11::arg("q"), pybind11::arg("k"),
          pybind11::arg("v"), pybind11::arg("log_decay"), pybind11::arg("scale"), pybind11::arg("initial_state") = pybind11::none(),
          pybind11::arg("return_last_state") = false, pybind11::arg("keep_states") = false);
    m.def("linattn_bwd", &linattn_bwd, "Linear attention backward [dq, dk, dv, dlog_decay?, dinitial_state?]", pybind11::arg("q"),
          pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("log_decay"), pybind11::arg("scale"), pybind11::arg("initial_state"),
          pybind11::arg("dout"), pybind11::arg("dlast_state"), pybind11::arg("states"), pybind11::arg("decay_per_head"), pybind11::arg("want_decay"),
          pybind11::arg("want_initial"));
    m.def("linattn_update", &linattn_update, "Linear attention, one token (in place on state)", pybind11::arg("state"), pybind11::arg("q"),
          pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("log_decay"), pybind11::arg("scale"));
    m.def("group_norm_fwd", &group_norm_fwd, "Gated group norm forward", pybind11::arg("x"), pybind11::arg("n_groups"),
          pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("z"), pybind11::arg("eps"), pybind11::arg("is_rms"),
          pybind11::arg("gate"));
    m.def("group_norm_bwd", &group_norm_bwd, "Gated group norm backward [dx, dweight?, dbias?, dz?]", pybind11::arg("x"),
          pybind11::arg("n_groups"), pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("z"), pybind11::arg("eps"),
          pybind11::arg("is_rms"), pybind11::arg("gate"), pybind11::arg("dout"), pybind11::arg("want_weights"));
    m.def("delta_fwd", &delta_fwd, "Gated delta rule forward [out, last_state?, states of the segments?]", pybind11::arg("q"), pybind11::arg("k"), pybind11::arg("v"),
          pybind11::arg("beta"), pybind11::arg("log_decay"), pybind11::arg("scale"), pybind11::arg("initial_state"), pybind11::arg("return_last_state"),
          pybind11::arg("keep_states"));
    m.def("delta_bwd", &delta_bwd, "Gated delta rule backward [dq, dk, dv, dbeta, dlog_decay?, dinitial_state?]", pybind11::arg("q"),
          pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("beta"), pybind11::arg("log_decay"), pybind11::arg("scale"),
          pybind11::arg("initial_state"), pybind11::arg("dout"), pybind11::arg("dlast_state"), pybind11::arg("states"),
          pybind11::arg("decay_per_head"), pybind11::arg("want_decay"), pybind11::arg("want_initial"));
    m.def("delta_update", &delta_update, "Gated delta rule, one token (in place on state)", pybind11::arg("state"), pybind11::arg("q"),
          pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("beta"), pybind11::arg("log_decay"), pybind11::arg("scale"));
    m.def("layer_norm_fwd", &layer_norm_fwd, "Residual add and layer norm forward [out, residual_out?]", pybind11::arg("x"),
          pybind11::arg("residual"), pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("eps"), pybind11::arg("is_rms"),
          pybind11::arg("want_residual"), pybind11::arg("wide"));
    m.def("layer_norm_bwd", &layer_norm_bwd, "Residual add and layer norm backward [dx?, dresidual?, dweight?, dbias?]", pybind11::arg("x"),
          pybind11::arg("residual"), pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("eps"), pybind11::arg("is_rms"),
          pybind11::arg("dout"), pybind11::arg("dresidual_out"), pybind11::arg("wide"), pybind11::arg("want_dx"), pybind11::arg("want_dresidual"),
          pybind11::arg("want_weight"), pybind11::arg("want_bias"));
    m.def("abi_version", []() { return mm_abi_version(); });
}
