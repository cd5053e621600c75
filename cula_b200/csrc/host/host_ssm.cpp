// The operators of a selective state space block (selective scan, single-token steps, residual RMS norm) on the native host path.
#include <algorithm>
#include <climits>

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include "host_common.h"

namespace cula_host {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t KEEP = 8;                    // tokens per kept state
constexpr int64_t SMS = 148;                   // of a B200: the models below were fitted there

bool grad_wanted(std::initializer_list<OptTensor> ts) {
    for (const OptTensor& t : ts)
        if (t.has_value() && has_tangent(*t)) return true;
    if (!at::GradMode::is_enabled()) return false;
    for (const OptTensor& t : ts)
        if (t.has_value() && t->defined() && t->requires_grad()) return true;
    return false;
}
// an operator without gradients: a tangent would be lost without a word
using cula_host::has_tangent;
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... Ts>
void refuse_tangents(const char* op, const Ts&... ts) {
    if ((has_tangent(ts) || ...)) throw std::runtime_error(std::string(op) + " has no forward derivative");
}
OptTensor opt_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
bool is_float(const Tensor& t) { return is_bf16(t) || is_f32(t); }
bool aligned(const Tensor& t, uintptr_t bytes = 16) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (bytes - 1)) == 0; }
void on_device_of(const Tensor& x, std::initializer_list<std::pair<OptTensor, const char*>> ts) {
    for (const auto& [t, name] : ts)
        if (has(t) && t->device() != x.device())
            throw pybind11::value_error(std::string(name) + " must be on the device of x (" + x.device().str() + "), not on " + t->device().str() + ".");
}
// contiguous fp32 whose first element is 16-byte aligned: the kernels read parameters in wide pieces
Tensor param(const Tensor& t) {
    Tensor c = contiguous_f32(t);
    return aligned(c) ? c : c.clone();
}
OptTensor param(const OptTensor& t) { return has(t) ? OptTensor(param(*t)) : OptTensor(); }
// Rows as the kernels take them: the innermost dimensions contiguous, 16-byte aligned rows. Views that fit (a part of a projection's
// output) are used in place, others are copied.
bool rows_fit(const Tensor& t, int64_t inner_dims, int64_t align_elements, uintptr_t align_bytes) {
    int64_t expect = 1;
    for (int64_t d = t.dim() - 1; d >= t.dim() - inner_dims; --d) {
        if (t.size(d) != 1 && t.stride(d) != expect) return false;
        expect *= t.size(d);
    }
    for (int64_t d = 0; d < t.dim() - inner_dims; ++d)
        if (t.size(d) != 1 && (t.stride(d) % align_elements || t.stride(d) > INT_MAX && d > 0)) return false;       // from token to token: 32 bits
    return aligned(t, align_bytes);
}
Tensor rows_of(const Tensor& t, int64_t inner_dims) {
    const int64_t align = inner_dims == 1 ? 16 / t.element_size() : 1;
    if (rows_fit(t, inner_dims, align, inner_dims == 1 ? 16 : t.element_size())) return t;
    return t.is_contiguous() ? t.clone() : t.contiguous();
}
long long stride_of(const Tensor& t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

// A backward pass that is captured into a graph while an eager graph of the same leaves lives on the default stream: their accumulators belong
// to that stream, the engine would wait on it across the capture, and that ends the process. Said here, before it happens. (Accumulators
// of other streams can be waited on.)
void refuse_accumulators_of_the_default_stream(const Tensor& like) {
    if (at::cuda::currentStreamCaptureStatus() == at::cuda::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const c10::Stream outside = c10::cuda::getDefaultCUDAStream(like.device().index()).unwrap();
    for (const auto& edge : node->next_edges())
        if (edge.function && dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get()))
            if (const auto stream = edge.function->stream(); stream.has_value() && *stream == outside)
                throw std::runtime_error("a backward pass cannot be captured while an earlier graph of the same leaves lives: its outputs hold their "
                                         "gradient accumulators, which belong to the default stream; let go of them first");
}

// Gradients that a graph is made of (create_graph) hang on the operator's inputs by a node that says that it cannot be differentiated:
// left as constants, they would give second derivatives with a part missing.
variable_list differentiable_once(variable_list grads) {
    const auto node = torch::autograd::get_current_node();
    if (!at::GradMode::is_enabled() || !node) return grads;
    torch::autograd::edge_list inputs = node->next_edges();
    const auto error = std::make_shared<torch::autograd::Error>("the gradients of this operator cannot be differentiated again", std::move(inputs));
    for (Tensor& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(g, error);
        }
    return grads;
}

// ------------------------------------------------ selective scan ------------------------------------------------
int64_t padded_states(int64_t S) { return S <= 8 ? 8 : S <= 16 ? 16 : S <= 32 ? 32 : 64; }

struct ScanInputs {
    Tensor x, dt, A, B, C;
    OptTensor skip, z, bias, h0;
    bool softplus = false;
    std::optional<Tables> tab;
};
struct ScanSizes {
    int64_t B, T, D, S, G, SP, n_seqs, num_chunks, longest, tiles;        // longest: chunks of the longest sequence; tiles: of channels
    bool packed;
};
ScanSizes sizes_of(const ScanInputs& in) {
    ScanSizes s{};
    s.B = in.x.size(0); s.T = in.x.size(1); s.D = in.x.size(2); s.G = in.B.size(2); s.S = in.B.size(3);
    s.SP = padded_states(s.S);
    s.packed = in.tab.has_value();
    const int64_t cps = (s.T + CHUNK - 1) / CHUNK;
    s.n_seqs = in.tab ? in.tab->n_seqs : s.B;
    s.num_chunks = in.tab ? in.tab->num_chunks : s.B * cps;
    s.longest = in.tab ? in.tab->longest : cps;
    s.tiles = lib.cula_kda_selective_scan_tiles((int)s.D, (int)s.G, (int)s.S) * s.G;
    return s;
}
// Microseconds that a CTA takes for a 64-token chunk of a tile of channels (16 states): alone on its SM, and beside another one
struct ScanCost { double alone, shared; };
// and what that model of a launch lacks, fitted to sweeps over segments: setting up a CTA, the last CTAs' share, a segment taken in
struct ScanFit { double set_up, tail, folded; };
// of a launch of so many CTAs of at most so many chunks each, `work` chunks in all
double scan_time(double ctas, double chunks, double work, ScanCost c, ScanFit f) {
    const double places = 2.0 * SMS, one = f.set_up + chunks * (ctas <= SMS ? c.alone : c.shared);
    return ctas <= places ? one : std::max(one, (work * c.shared + f.set_up * ctas) / places) + f.tail * one;
}
// Chunks per segment, 0 for sequences in one piece. Cutting takes a launch more, which makes the exponentials of nearly all tokens once
// more, and pays where few or long sequences would leave SMs waiting. Measured (whole, cut; us): 1 x 4096 tokens x 4096 channels forward
// 266, 191, backward 725, 373; 1 x 16384 x 512 forward 1038, 115, backward 2775, 225; 2 x 4096 x 4096 forward 266, 358 (whole), 20 packed
// sequences of 8192 in all x 2048 forward 152, 178 (whole), backward 549, 356; 1 x 512 x 4096 forward 39, 33.
int64_t plan_segments(const ScanSizes& s, bool backward) {
    const ScanCost walk = backward ? ScanCost{11.3, 17.7} : ScanCost{4.3, 7.0}, first = backward ? ScanCost{4.0, 5.2} : ScanCost{3.0, 5.2};
    const ScanFit fit = backward ? ScanFit{1.0, 0.25, 0.12} : ScanFit{2.0, 0.15, 0.03};
    const double tiles = (double)s.tiles, work = (double)s.num_chunks * tiles, longest = (double)s.longest;
    // whole: the longest sequence, beside others for as much of its time as there is work for the places beside it
    const double beside = std::min(1.0, work / (2.0 * SMS * std::max(1.0, longest)));
    double best = std::max((double)s.n_seqs * tiles <= SMS ? longest * walk.alone : longest * (walk.alone + beside * (walk.shared - walk.alone)),
                           work * walk.shared / (2.0 * SMS));
    int64_t seg = 0;
    for (int64_t k = 1; k < s.longest; k += (k + 3) / 4) {
        const double per_seq = std::ceil(longest / k), pieces = s.packed ? s.num_chunks / (double)k + 0.5 * s.n_seqs : s.n_seqs * per_seq, ctas = pieces * tiles;
        const double folded = fit.folded * per_seq * std::max(1.0, ctas / (2.0 * SMS));
        const double time = scan_time(ctas, (double)k, work, walk, fit) + scan_time(ctas, (double)k, work, first, fit) + 2.0 + folded;
        if (time < 0.95 * best) {
            best = time;
            seg = k;
        }
    }
    return seg;
}
int64_t segment_slots(const ScanSizes& s, const ScanInputs& in, int64_t seg) {
    if (!seg) return 0;
    return in.tab ? s.num_chunks / seg + s.n_seqs : s.n_seqs * ((s.longest + seg - 1) / seg);
}
cula_kda_selective_scan_args scan_args(const ScanInputs& in, const ScanSizes& s) {
    cula_kda_selective_scan_args a{};
    a.x = ptr(in.x); a.dt = ptr(in.dt); a.z = ptr(in.z); a.Bm = ptr(in.B); a.Cm = ptr(in.C);
    a.x_row = stride_of(in.x, 1); a.x_seq = stride_of(in.x, 0);
    a.dt_row = stride_of(in.dt, 1); a.dt_seq = stride_of(in.dt, 0);
    if (has(in.z)) { a.z_row = stride_of(*in.z, 1); a.z_seq = stride_of(*in.z, 0); }
    a.b_row = stride_of(in.B, 1); a.b_seq = stride_of(in.B, 0);
    a.c_row = stride_of(in.C, 1); a.c_seq = stride_of(in.C, 0);
    a.A = fptr(in.A); a.skip = fptr(in.skip); a.dt_bias = fptr(in.bias); a.h0 = fptr(in.h0);
    if (in.tab) {
        a.cu_seqlens = (int*)ptr(in.tab->cu_seqlens); a.chunk_indices = (int*)ptr(in.tab->chunk_indices);
        a.chunk_offsets = (int*)ptr(in.tab->chunk_offsets); a.seq_order = (int*)ptr(in.tab->seq_order);
        a.total_tokens = (int)in.tab->total_tokens;
    }
    a.rows = s.B * s.T; a.T = (int)s.T; a.D = (int)s.D; a.S = (int)s.S; a.G = (int)s.G; a.n_seqs = (int)s.n_seqs; a.num_chunks = (int)s.num_chunks;
    a.softplus = in.softplus; a.fp32 = is_f32(in.x);
    const uintptr_t quad = 4 * in.B.element_size();
    a.vec_bc = (s.S % 4 == 0 || s.G == 1) && a.b_row % 4 == 0 && a.b_seq % 4 == 0 && a.c_row % 4 == 0 && a.c_seq % 4 == 0 && aligned(in.B, quad) && aligned(in.C, quad);
    return a;
}
struct ScanOutputs {
    Tensor y, hT, states, y_pre;
};
bool no_token(const ScanInputs& in) { return in.x.numel() == 0 || (in.tab && in.tab->total_tokens == 0); }
ScanOutputs scan_forward(const ScanInputs& in, bool want_final, bool keep) {
    c10::cuda::CUDAGuard guard(in.x.device());
    const ScanSizes s = sizes_of(in);
    const auto f32 = in.A.options();
    ScanOutputs o;
    if (no_token(in)) {                                              // the states stay what they were
        o.y = at::zeros({s.B, s.T, s.D}, in.x.options());
        if (want_final) o.hT = has(in.h0) ? in.h0->clone() : at::zeros({s.n_seqs, s.D, s.S}, f32);
        return o;
    }
    o.y = device_empty({s.B, s.T, s.D}, in.x.options());
    if (in.tab && in.tab->total_tokens < s.T) o.y.narrow(1, in.tab->total_tokens, s.T - in.tab->total_tokens).zero_();      // rows past the packed tokens
    if (want_final) o.hT = device_empty({s.n_seqs, s.D, s.S}, f32);
    if (keep) {
        o.states = device_empty({s.num_chunks * (CHUNK / KEEP), lib.cula_kda_selective_scan_state_floats((int)s.D, (int)s.G, (int)s.S)}, f32);
        if (has(in.z)) o.y_pre = device_empty({s.B, s.T, s.D}, f32);
    }
    cula_kda_selective_scan_args a = scan_args(in, s);
    a.y = ptr(o.y); a.hT = fptr(o.hT); a.states = fptr(o.states); a.y_pre = fptr(o.y_pre);
    a.seg_chunks = (int)plan_segments(s, false);
    Tensor seg;
    if (a.seg_chunks) {
        const int64_t n = segment_slots(s, in, a.seg_chunks);
        seg = device_empty({n * s.D * (s.SP + 1)}, f32);
        a.seg_state = fptr(seg);
        a.seg_dt = a.seg_state + n * s.D * s.SP;
    }
    check(lib.cula_kda_selective_scan_fwd(&a, stream_of(in.x)), "cula_kda_selective_scan_fwd");
    return o;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                 const OptTensor& skip, const OptTensor& z, const OptTensor& bias, const OptTensor& h0, bool softplus, bool want_final,
                                 const Tables* tab) {
        ScanInputs in{rows_of(x, 1), rows_of(dt, 1), param(A), rows_of(B, 2), rows_of(C, 2), param(skip), has(z) ? OptTensor(rows_of(*z, 1)) : OptTensor(),
                      param(bias), has(h0) ? OptTensor(h0->contiguous()) : OptTensor(), softplus, tab ? std::optional<Tables>(*tab) : std::nullopt};
        ScanOutputs o = scan_forward(in, want_final, true);
        ctx->save_for_backward({in.x, in.dt, in.A, in.B, in.C, in.skip.value_or(Tensor()), in.z.value_or(Tensor()), in.bias.value_or(Tensor()), o.states, o.y_pre});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["h0"] = has(h0) && h0->requires_grad();
        if (tab) {
            ctx->saved_data["tab"] = std::vector<Tensor>{tab->cu_seqlens, tab->chunk_indices, tab->chunk_offsets, tab->seq_order};
            ctx->saved_data["tab_sizes"] = std::vector<int64_t>{tab->n_seqs, tab->num_chunks, tab->total_tokens, tab->longest};
        }
        ctx->set_materialize_grads(false);
        if (!want_final) return {o.y};
        return {o.y, o.hT};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(12);
        const Tensor dhT = grads.size() > 1 && grads[1].defined() ? contiguous_f32(grads[1]) : Tensor();
        if (!grads[0].defined() && !dhT.defined()) return out;
        auto v = ctx->get_saved_variables();
        refuse_accumulators_of_the_default_stream(v[0]);
        ScanInputs in{v[0], v[1], v[2], v[3], v[4], opt_of(v[5]), opt_of(v[6]), opt_of(v[7]), OptTensor(), ctx->saved_data["softplus"].toBool(), std::nullopt};
        if (auto it = ctx->saved_data.find("tab"); it != ctx->saved_data.end()) {
            auto t = it->second.toTensorVector();
            auto n = ctx->saved_data["tab_sizes"].toIntVector();
            in.tab = Tables{t[0], t[1], t[2], t[3], n[0], n[1], n[2], n[3]};
        }
        c10::cuda::CUDAGuard guard(in.x.device());
        const cudaStream_t stream = stream_of(in.x);
        const ScanSizes s = sizes_of(in);
        const auto f32 = in.A.options(), act = in.x.options();
        if (no_token(in)) {
            auto none = [&](const OptTensor& t) { return has(t) ? at::zeros(t->sizes(), t->options()) : Tensor(); };
            const Tensor dh0 = !ctx->saved_data["h0"].toBool() ? Tensor() : dhT.defined() ? dhT.clone() : at::zeros({s.n_seqs, s.D, s.S}, f32);
            return differentiable_once({none(in.x), none(in.dt), none(in.A), none(in.B), none(in.C), none(in.skip), none(in.z), none(in.bias), dh0,
                                        Tensor(), Tensor(), Tensor()});
        }
        Tensor dy;
        if (grads[0].defined()) {
            dy = grads[0].contiguous();
            if (dy.scalar_type() != in.x.scalar_type()) dy = dy.to(in.x.scalar_type());
            if (!aligned(dy)) dy = dy.clone();
        } else dy = device_empty({s.B, s.T, s.D}, act).zero_();
        cula_kda_selective_scan_args a = scan_args(in, s);
        Tensor dx = device_empty({s.B, s.T, s.D}, act), ddt = device_empty({s.B, s.T, s.D}, act), dz;
        if (has(in.z)) dz = device_empty({s.B, s.T, s.D}, act);
        if (in.tab && in.tab->total_tokens < s.T)
            for (Tensor* t : {&dx, &ddt, &dz})
                if (t->defined()) t->narrow(1, in.tab->total_tokens, s.T - in.tab->total_tokens).zero_();
        Tensor dB = device_empty({s.B, s.T, s.G, s.S}, act), dC = device_empty({s.B, s.T, s.G, s.S}, act);
        Tensor dA = device_empty({s.D, s.S}, f32), dskip, dbias, dh0;
        if (has(in.skip)) dskip = device_empty(in.skip->sizes(), f32);
        if (has(in.bias)) dbias = device_empty(in.bias->sizes(), f32);
        if (ctx->saved_data["h0"].toBool()) dh0 = device_empty({s.n_seqs, s.D, s.S}, f32);
        a.states = fptr(v[8]); a.y_pre = fptr(v[9]); a.dy = ptr(dy); a.dhT = fptr(dhT);
        a.dx = ptr(dx); a.ddt = ptr(ddt); a.dz = ptr(dz); a.dBm = ptr(dB); a.dCm = ptr(dC);
        a.dA = fptr(dA); a.dskip = fptr(dskip); a.dbias = fptr(dbias); a.dh0 = fptr(dh0);
        a.seg_chunks = (int)plan_segments(s, true);
        const int64_t n_seg = segment_slots(s, in, a.seg_chunks);
        const int64_t items = a.seg_chunks ? n_seg : s.n_seqs;
        a.cta_rows = (int)std::max<int64_t>(1, std::min(items, 8 * SMS / s.tiles));
        // one workspace: shares of dB and dC, of dA, dskip and dbias, segments
        const int64_t n_bc = s.tiles / s.G * a.rows * s.G * 2 * s.SP, n_A = a.cta_rows * s.D * (s.SP + 2);
        Tensor work = device_empty({n_bc + n_A + n_seg * s.D * (s.SP + 1)}, f32);
        a.part_bc = fptr(work);
        a.part_A = a.part_bc + n_bc;
        a.part_skip = has(in.skip) ? a.part_A + a.cta_rows * s.D * s.SP : nullptr;
        a.part_bias = has(in.bias) ? a.part_A + a.cta_rows * s.D * (s.SP + 1) : nullptr;
        if (a.seg_chunks) {
            a.seg_state = a.part_A + n_A;
            a.seg_dt = a.seg_state + n_seg * s.D * s.SP;
        }
        check(lib.cula_kda_selective_scan_bwd(&a, stream), "cula_kda_selective_scan_bwd");
        return differentiable_once({dx, ddt, dA, dB, dC, dskip, dz, dbias, dh0, Tensor(), Tensor(), Tensor()});
    }
};

// [B, T, S] or [B, T, G, S] as the latter
Tensor grouped(const Tensor& m, int64_t full) { return m.dim() == full - 1 ? m.unsqueeze(-2) : m; }

void check_params(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip, const OptTensor& z,
                  const OptTensor& bias, int64_t lead) {
    const int64_t D = x.size(-1);
    require(is_float(x), "x must be in bfloat16 or float32.");
    require(dt.sizes() == x.sizes() && (!has(z) || z->sizes() == x.sizes()), "dt and z must have the shape of x.");
    require(dt.scalar_type() == x.scalar_type() && B.scalar_type() == x.scalar_type() && C.scalar_type() == x.scalar_type() &&
                (!has(z) || z->scalar_type() == x.scalar_type()), "dt, B, C and z must have the type of x.");
    require(A.dim() == 2 && A.size(0) == D && A.is_floating_point(), "A must be [D, S].");
    require(1 <= A.size(1) && A.size(1) <= 64, "the state size must be 1 to 64.");
    require(B.dim() == lead + 2 && C.sizes() == B.sizes() && B.size(-1) == A.size(1), "B and C must be [..., S] or [..., G, S] with the state size of A.");
    for (int64_t d = 0; d < lead; ++d) require(B.size(d) == x.size(d), "B and C must have the tokens of x.");
    const int64_t G = B.size(-2);
    require(D > 0 && G > 0 && D % G == 0 && D / G % 8 == 0, "the channels of each group of B and C must be a multiple of 8.");
    require(!has(skip) || (skip->dim() == 1 && skip->size(0) == D), "D must be [D].");
    require(!has(bias) || (bias->dim() == 1 && bias->size(0) == D), "dt_bias must be [D].");
    on_device_of(x, {{dt, "dt"}, {A, "A"}, {B, "B"}, {C, "C"}, {skip, "D"}, {z, "z"}, {bias, "dt_bias"}});
}

std::pair<Tensor, OptTensor> selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B_in, const Tensor& C_in, const OptTensor& skip,
                                            const OptTensor& z, const OptTensor& bias, bool softplus, const OptTensor& h0, bool want_final, const Tables* tab) {
    require(x.dim() == 3, "x must be [B, T, D].");
    require((B_in.dim() == 3 || B_in.dim() == 4) && B_in.dim() == C_in.dim(), "B and C must be [B, T, S] or [B, T, G, S].");
    const Tensor B = grouped(B_in, 4), C = grouped(C_in, 4);
    check_params(x, dt, A, B, C, skip, z, bias, 2);
    if (tab) {
        if (x.size(0) != 1)
            throw pybind11::value_error("The batch size is expected to be 1 rather than " + std::to_string(x.size(0)) + " when using `cu_seqlens`.");
        if (tab->total_tokens > x.size(1))
            throw pybind11::value_error("cu_seqlens ends at " + std::to_string(tab->total_tokens) + ", past the " + std::to_string(x.size(1)) + " tokens of x.");
        on_device_of(x, {{tab->cu_seqlens, "cu_seqlens"}});
    }
    const int64_t n_seqs = tab ? tab->n_seqs : x.size(0), D = x.size(2), S = A.size(1);
    if (has(h0)) {
        if (h0->dim() != 3 || h0->size(0) != n_seqs || h0->size(1) != D || h0->size(2) != S)
            throw pybind11::value_error("initial_state must be [" + std::to_string(n_seqs) + ", " + std::to_string(D) + ", " + std::to_string(S) + "].");
        require(is_f32(*h0), "initial_state must be in float32.");
        on_device_of(x, {{h0, "initial_state"}});
    }
    require(x.size(1) <= (int64_t)1 << 30 && x.size(0) <= (int64_t)1 << 30 && D <= (int64_t)1 << 24, "too many tokens or channels.");
    assert_blackwell(x);
    if (grad_wanted({x, dt, A, B, C, skip, z, bias, h0})) {
        auto out = SelectiveScan::apply(x, dt, A, B, C, skip, z, bias, h0, softplus, want_final, tab);
        return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
    }
    at::NoGradGuard no_grad;
    const ScanInputs in{rows_of(x, 1), rows_of(dt, 1), param(A), rows_of(B, 2), rows_of(C, 2), param(skip), has(z) ? OptTensor(rows_of(*z, 1)) : OptTensor(),
                        param(bias), has(h0) ? OptTensor(h0->contiguous()) : OptTensor(), softplus, tab ? std::optional<Tables>(*tab) : std::nullopt};
    ScanOutputs o = scan_forward(in, want_final, false);
    return {o.y, opt_of(o.hT)};
}

// ------------------------------------------------ single tokens ------------------------------------------------
// [N, ...] or [N, 1, ...] as the former
Tensor one_token(const Tensor& t, bool with_time) { return with_time ? t.squeeze(1) : t; }

// The slots of a call: int32 on the device. A pool without indices holds one state per sequence.
OptTensor slots_of(const OptTensor& indices, const Tensor& x, int64_t rows, int64_t pool, const char* name) {
    if (!has(indices)) {
        if (pool < rows)
            throw pybind11::value_error("the pool holds " + std::to_string(pool) + " states for " + std::to_string(rows) + " sequences and no indices were given");
        return OptTensor();
    }
    if (indices->dim() != 1 || indices->size(0) != rows || (indices->scalar_type() != at::kInt && indices->scalar_type() != at::kLong))
        throw pybind11::value_error(std::string(name) + " must hold one int32 slot per sequence");
    on_device_of(x, {{indices, name}});
    if (indices->scalar_type() == at::kInt) return indices->contiguous();
    return indices->clamp(-1, INT_MAX).to(at::kInt).contiguous();            // what is past 32 bits is past the pool, not another slot
}
void check_out(const OptTensor& out, const Tensor& x) {
    if (!has(out)) return;
    if (out->sizes() != x.sizes() || out->scalar_type() != x.scalar_type() || !out->is_contiguous() || !aligned(*out))
        throw pybind11::value_error("out must be a contiguous, 16-byte aligned tensor of the shape and type of x");
    on_device_of(x, {{out, "out"}});
}
// autograd learns that a tensor was written to: a graph that has kept it must not take it for what it was
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor output_of(const OptTensor& out, const Tensor& x) { return has(out) ? *out : device_empty(x.sizes(), x.options()); }

Tensor selective_scan_update(const Tensor& x_in, const Tensor& dt_in, const Tensor& A_in, const Tensor& B_in, const Tensor& C_in, const Tensor& state,
                             const OptTensor& indices, const OptTensor& skip_in, const OptTensor& z_in, const OptTensor& bias_in, bool softplus,
                             const OptTensor& out_in) {
    refuse_tangents("selective_scan_update", x_in, dt_in, A_in, B_in, C_in, state, skip_in, z_in, bias_in);
    at::NoGradGuard no_grad;
    const bool with_time = x_in.dim() == 3;
    require(x_in.dim() == 2 || (with_time && x_in.size(1) == 1), "x must be [N, D] or [N, 1, D].");
    require(dt_in.sizes() == x_in.sizes() && (!has(z_in) || z_in->sizes() == x_in.sizes()), "dt and z must have the shape of x.");
    const int64_t lead = with_time ? 2 : 1;
    require((B_in.dim() == lead + 1 || B_in.dim() == lead + 2) && B_in.dim() == C_in.dim() && (!with_time || (B_in.size(1) == 1 && C_in.size(1) == 1)),
            "B and C must be [N, S] or [N, G, S], with the token axis of x.");
    const Tensor x = one_token(x_in, with_time), dt = one_token(dt_in, with_time);
    const OptTensor z = has(z_in) ? OptTensor(one_token(*z_in, with_time)) : OptTensor();
    const Tensor B = grouped(one_token(B_in, with_time), 3), C = grouped(one_token(C_in, with_time), 3);
    check_params(x, dt, A_in, B, C, skip_in, z, bias_in, 1);
    const int64_t N = x.size(0), D = x.size(1), G = B.size(1), S = B.size(2);
    if (state.dim() != 3 || state.size(1) != D || state.size(2) != S)
        throw pybind11::value_error("state must be [pool, " + std::to_string(D) + ", " + std::to_string(S) + "].");
    require(is_f32(state) && state.is_contiguous(), "the state pool must be contiguous float32");
    on_device_of(x, {{state, "state"}});
    require(N <= (int64_t)1 << 24 && D <= (int64_t)1 << 24 && state.size(0) <= (int64_t)1 << 30, "too many sequences, channels or states.");
    const OptTensor idx = slots_of(indices, x, N, state.size(0), "state_indices");
    check_out(out_in, x_in);
    assert_blackwell(x);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor out = output_of(out_in, x_in);
    if (N == 0) return out;
    auto rows = [](const Tensor& t, int64_t inner) { return rows_fit(t, inner, 1, t.element_size()) ? t : t.contiguous(); };
    const Tensor xr = rows(x, 1), dtr = rows(dt, 1), Br = rows(B, 2), Cr = rows(C, 2), A = param(A_in);
    const OptTensor zr = has(z) ? OptTensor(rows(*z, 1)) : OptTensor(), skip = contiguous_f32(skip_in), bias = contiguous_f32(bias_in);
    cula_kda_selective_step_args a{};
    a.x = ptr(xr); a.dt = ptr(dtr); a.z = ptr(zr); a.Bm = ptr(Br); a.Cm = ptr(Cr);
    a.A = fptr(A); a.skip = fptr(skip); a.dt_bias = fptr(bias); a.state = fptr(state); a.indices = iptr(idx); a.y = ptr(out);
    a.x_row = stride_of(xr, 0); a.dt_row = stride_of(dtr, 0); a.z_row = has(zr) ? stride_of(*zr, 0) : 0; a.b_row = stride_of(Br, 0); a.c_row = stride_of(Cr, 0);
    a.rows = (int)N; a.D = (int)D; a.S = (int)S; a.G = (int)G; a.pool = (int)state.size(0); a.softplus = softplus; a.fp32 = is_f32(x);
    const uintptr_t quad = 4 * Br.element_size();
    a.vec = S % 4 == 0 && a.b_row % 4 == 0 && a.c_row % 4 == 0 && aligned(Br, quad) && aligned(Cr, quad) && aligned(state);
    a.status = status_word(x.device().index());
    check(lib.cula_kda_selective_step(&a, stream_of(x)), "cula_kda_selective_step");
    written(state);
    if (has(out_in)) written(out);
    return out;
}

Tensor short_conv_update(const Tensor& x_in, const Tensor& weight_in, const Tensor& cache, const OptTensor& indices, const OptTensor& bias_in, bool silu,
                         const OptTensor& out_in) {
    refuse_tangents("short_conv_update", x_in, weight_in, cache, bias_in);
    at::NoGradGuard no_grad;
    const bool with_time = x_in.dim() == 3;
    require((x_in.dim() == 2 || (with_time && x_in.size(1) == 1)) && is_bf16(x_in), "x must be [N, D] or [N, 1, D] in bfloat16.");
    const Tensor x = one_token(x_in, with_time);
    require(weight_in.dim() == 2 || (weight_in.dim() == 3 && weight_in.size(1) == 1), "weight must be [D, W] with W <= 4 and D a multiple of 8.");
    const Tensor weight = weight_in.dim() == 3 ? weight_in.squeeze(1) : weight_in;
    const int64_t N = x.size(0), D = weight.size(0), W = weight.size(1);
    require(x.size(1) == D && D > 0 && D % 8 == 0 && 1 <= W && W <= 4, "weight must be [D, W] with W <= 4 and D a multiple of 8.");
    require(!has(bias_in) || bias_in->numel() == D, "bias must be [D].");
    if (cache.dim() != 3 || cache.size(1) != D || cache.size(2) != W)
        throw pybind11::value_error("cache must be [pool, " + std::to_string(D) + ", " + std::to_string(W) + "].");
    require(is_f32(cache) && cache.is_contiguous(), "the pool of windows must be contiguous float32");
    on_device_of(x, {{weight, "weight"}, {cache, "cache"}, {bias_in, "bias"}});
    require(N <= (int64_t)1 << 24 && D <= (int64_t)1 << 24 && cache.size(0) <= (int64_t)1 << 30, "too many sequences, channels or windows.");
    const OptTensor idx = slots_of(indices, x, N, cache.size(0), "cache_indices");
    check_out(out_in, x_in);
    if (!aligned(cache)) throw pybind11::value_error("the pool of windows must be 16-byte aligned");
    assert_blackwell(x);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor out = output_of(out_in, x_in);
    if (N == 0) return out;
    const Tensor xr = rows_fit(x, 1, 2, 4) ? x : x.is_contiguous() ? x.clone() : x.contiguous(), w = param(weight);
    const OptTensor bias = contiguous_f32(bias_in);
    cula_kda_conv_step_args a{};
    a.x = ptr(xr); a.w = fptr(w); a.bias = fptr(bias); a.cache = fptr(cache); a.indices = iptr(idx); a.y = ptr(out); a.x_row = stride_of(xr, 0);
    a.rows = (int)N; a.D = (int)D; a.W = (int)W; a.pool = (int)cache.size(0); a.silu = silu;
    a.status = status_word(x.device().index());
    check(lib.cula_kda_conv_step(&a, stream_of(x)), "cula_kda_conv_step");
    written(cache);
    if (has(out_in)) written(out);
    return out;
}

// ------------------------------------------------ residual RMS norm ------------------------------------------------
int res_code(const OptTensor& r) { return !has(r) ? 0 : is_bf16(*r) ? 1 : 2; }

// rows of a norm: two-dimensional views are used in place
Tensor norm_rows(const Tensor& t) {
    if (t.dim() == 2 && rows_fit(t, 1, 16 / t.element_size(), 16)) return t;
    const Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}
long long row_stride(const Tensor& t) { return t.dim() == 2 ? stride_of(t, 0) : t.size(-1); }

struct NormOutputs {
    Tensor y, r_out, rstd, scale;
};
NormOutputs add_norm_forward(const Tensor& x, const OptTensor& r, const Tensor& w, double eps, bool keep, bool fp8, int64_t group) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t D = x.size(-1), R = x.numel() / D;
    const auto f32 = x.options().dtype(at::kFloat);
    NormOutputs o;
    o.y = device_empty(x.sizes(), fp8 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
    if (has(r)) o.r_out = device_empty(r->sizes(), r->options());
    if (keep) o.rstd = device_empty({R}, f32);
    if (fp8) {
        auto shape = x.sizes().vec();
        if (group) shape.back() = D / group;
        else shape.pop_back();
        o.scale = device_empty(shape, f32);
    }
    if (R == 0) return o;
    cula_kda_add_rms_norm_args a{};
    a.x = ptr(x); a.r = ptr(r); a.w = fptr(w); a.y = ptr(o.y); a.r_out = ptr(o.r_out); a.rstd = fptr(o.rstd); a.scale = fptr(o.scale);
    a.R = R; a.D = (int)D; a.x_row = row_stride(x); a.r_row = has(r) ? row_stride(*r) : 0; a.group = (int)group;
    a.fp32 = is_f32(x); a.res = res_code(r); a.fp8 = fp8; a.eps = (float)eps;
    check(lib.cula_kda_add_rms_norm_fwd(&a, stream_of(x)), "cula_kda_add_rms_norm_fwd");
    return o;
}

struct AddNorm : torch::autograd::Function<AddNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x_in, const OptTensor& r_in, const Tensor& weight, double eps) {
        const Tensor x = norm_rows(x_in), w = param(weight);
        const OptTensor r = has(r_in) ? OptTensor(norm_rows(*r_in)) : OptTensor();
        NormOutputs o = add_norm_forward(x, r, w, eps, true, false, 0);
        ctx->save_for_backward({has(r) ? o.r_out : x, w, o.rstd});   // the sum that was kept is all that the backward pass needs
        ctx->saved_data["res"] = (int64_t)res_code(r);
        ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
        ctx->set_materialize_grads(false);
        if (!has(r)) return {o.y};
        return {o.y, o.r_out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool with_r = grads.size() > 1;
        if (!grads[0].defined() && (!with_r || !grads[1].defined())) return variable_list(4);
        auto s = ctx->get_saved_variables();
        const Tensor &v = s[0], &w = s[1], &rstd = s[2];
        refuse_accumulators_of_the_default_stream(v);
        const auto x_type = (at::ScalarType)ctx->saved_data["x_type"].toInt();
        const int64_t res = ctx->saved_data["res"].toInt(), D = v.size(-1), R = v.numel() / D;
        c10::cuda::CUDAGuard guard(v.device());
        auto upstream = [&](const Tensor& g, at::ScalarType type) {
            Tensor t = g.scalar_type() == type ? g.contiguous() : g.to(type).contiguous();
            return aligned(t) ? t : t.clone();
        };
        Tensor dy = grads[0].defined() ? upstream(grads[0], x_type) : at::zeros(v.sizes(), v.options().dtype(x_type));
        Tensor dr_out = with_r && grads[1].defined() ? upstream(grads[1], v.scalar_type()) : Tensor();
        Tensor dx = device_empty(v.sizes(), v.options().dtype(x_type)), dr;
        if (res && v.scalar_type() != x_type) dr = device_empty(v.sizes(), v.options());
        Tensor dw = device_empty({D}, w.options());
        if (R == 0) return differentiable_once({dx, res ? (dr.defined() ? dr : dx) : Tensor(), dw.zero_(), Tensor()});
        Tensor part = device_empty({lib.cula_kda_add_rms_norm_shares((int)D, R), D}, w.options());
        cula_kda_add_rms_norm_args a{};
        a.v = ptr(v); a.w = fptr(w); a.rstd = fptr(rstd); a.dy = ptr(dy); a.dr_out = ptr(dr_out); a.dx = ptr(dx); a.dr = ptr(dr);
        a.part_w = fptr(part); a.dw = fptr(dw); a.R = R; a.D = (int)D; a.x_row = res ? D : row_stride(v);
        a.fp32 = x_type == at::kFloat; a.res = (int)res;
        check(lib.cula_kda_add_rms_norm_bwd(&a, stream_of(v)), "cula_kda_add_rms_norm_bwd");
        return differentiable_once({dx, res ? (dr.defined() ? dr : dx) : Tensor(), dw, Tensor()});
    }
};

void check_norm(const Tensor& x, const OptTensor& r, const Tensor& weight) {
    require(x.dim() >= 1 && is_float(x), "x must be in bfloat16 or float32.");
    const int64_t D = x.size(-1);
    require(D > 0 && D % 8 == 0 && D <= 16384, "the normalised dim must be a multiple of 8 up to 16384.");
    require(weight.dim() == 1 && weight.size(0) == D && weight.is_floating_point(), "weight must be [D].");
    if (has(r)) {
        require(r->sizes() == x.sizes(), "residual must have the shape of x.");
        require(is_float(*r) && (is_f32(*r) || is_bf16(x)), "residual must be in float32 or in the type of x.");
    }
    on_device_of(x, {{r, "residual"}, {weight, "weight"}});
    assert_blackwell(x);
}
std::pair<Tensor, OptTensor> add_rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& r, double eps) {
    check_norm(x, r, weight);
    if (grad_wanted({x, weight, r})) {
        auto out = AddNorm::apply(x, r, weight, eps);
        return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
    }
    at::NoGradGuard no_grad;
    NormOutputs o = add_norm_forward(norm_rows(x), has(r) ? OptTensor(norm_rows(*r)) : OptTensor(), param(weight), eps, false, false, 0);
    return {o.y, opt_of(o.r_out)};
}
std::tuple<Tensor, Tensor, OptTensor> add_rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& r, double eps, int64_t group) {
    refuse_tangents("add_rms_norm_fp8", x, weight, r);
    if (group) {
        require(group == 32 || group == 64 || group == 128 || group == 256, "group_size must be 32, 64, 128, 256 or None.");
        require(x.dim() >= 1 && x.size(-1) % group == 0, "the normalised dim must be a multiple of group_size.");
    }
    check_norm(x, r, weight);
    at::NoGradGuard no_grad;
    NormOutputs o = add_norm_forward(norm_rows(x), has(r) ? OptTensor(norm_rows(*r)) : OptTensor(), param(weight), eps, false, true, group);
    return {o.y, o.scale, opt_of(o.r_out)};
}

}  // namespace

void bind_ssm(pybind11::module_& m) {
    m.def("selective_scan", &selective_scan);
    // the planner alone: chunks per segment for so many sequences and chunks, the longest sequence's, and tiles of channels; 0: not cut
    m.def("selective_scan_segments", [](int64_t n_seqs, int64_t num_chunks, int64_t longest, int64_t tiles, bool packed, bool backward) {
        ScanSizes s{};
        s.n_seqs = n_seqs; s.num_chunks = num_chunks; s.longest = longest; s.tiles = tiles; s.packed = packed;
        return plan_segments(s, backward);
    });
    m.def("selective_scan_update", &selective_scan_update);
    m.def("short_conv_update", &short_conv_update);
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
}

}  // namespace cula_host
