// Operator Calls of a module: qk_norm_rope, attention and
// shared_prefix_attention. Their operands are buffers by name, their options
// numbers by name; everything the kernels assume of either is checked here,
// before any device work.
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <utility>
#include <vector>

#include "planner.h"

namespace mlk::hip {

namespace {

constexpr const char* kSlotNames[kOperandSlots] = {
    "q",          "k",       "v",          "prefix_k", "prefix_v", "q_weight", "k_weight", "positions", "slots", "q_offsets",
    "kv_start",   "kv_len",  "prefix_len", "q_out",    "k_out",    "v_out",    "out",      "lse"};

constexpr int64_t kMaxRows = INT32_MAX;   // rows are named by i32 buffers
constexpr int kMaxDim = 256, kMaxHeads = 4096;

int operandCode(Dtype d) {
    switch (d) {
        case Dtype::F32: return MLKD_F32;
        case Dtype::F16: return MLKD_F16;
        case Dtype::BF16: return MLKD_BF16;
        case Dtype::I32: return MLKD_I32;
        default: return MLKD_F64;
    }
}

/// One Call being read: its operands and attributes taken by name.
class Reader {
public:
    Reader(const KernelModule& km, const KernelNode& n) : km_(km), n_(n), what_(mathOpName(n.math)) {}

    const std::string& why() const { return why_; }
    bool fail(const std::string& m) {
        if (why_.empty()) why_ = what_ + ": " + m;
        return false;
    }

    /// Every name the Call holds is one of the given slots, with a buffer of
    /// its own that callers bind, or one of the given attributes.
    bool names(std::initializer_list<int> slots, std::initializer_list<const char*> attrs) {
        for (size_t i = 0; i < n_.operands.size(); ++i) {
            const auto& [name, id] = n_.operands[i];
            bool known = false;
            for (const int s : slots) known = known || name == kSlotNames[s];
            if (!known) return fail("unknown operand '" + name + "'");
            for (size_t j = 0; j < i; ++j) {
                if (n_.operands[j].first == name) return fail("operand '" + name + "' is given twice");
            }
            if (id >= km_.buffers.size()) return fail("operand '" + name + "' names no buffer");
            const KernelBuffer& b = km_.buffers[id];
            if (b.isTemp || (!b.isInput && !b.isOutput)) {
                return fail("operand '" + name + "' is neither an input nor an output");
            }
            if (b.dims.empty()) return fail("operand '" + name + "' has no dims");
            int64_t total = 1;   // of the dims that are not 0, so that every part of the product fits
            for (const int64_t d : b.dims) {
                if (d < 0 || (d > 0 && total > (int64_t{1} << 44) / d)) return fail("operand '" + name + "' is too large");
                total *= std::max<int64_t>(d, 1);
            }
        }
        for (size_t i = 0; i < n_.attrs.size(); ++i) {
            const std::string& name = n_.attrs[i].first;
            bool known = false;
            for (const char* a : attrs) known = known || name == a;
            // "<operand>_at" for the operands that are rows of heads.
            for (const int s : slots) known = known || (rowsOfHeads(s) && name == std::string(kSlotNames[s]) + "_at");
            if (!known) return fail("unknown attribute '" + name + "'");
            for (size_t j = 0; j < i; ++j) {
                if (n_.attrs[j].first == name) return fail("attribute '" + name + "' is given twice");
            }
        }
        return true;
    }

    bool has(int slot) const { return id(slot) != kInvalidId; }
    uint32_t id(int slot) const {
        for (const auto& [name, b] : n_.operands) {
            if (name == kSlotNames[slot]) return b;
        }
        return kInvalidId;
    }
    Dtype dtype(int slot) const { return km_.buffers[id(slot)].dtype; }

    bool real(const char* name, double fallback, double& v) {
        v = fallback;
        for (const auto& [key, value] : n_.attrs) {
            if (key == name) v = value;
        }
        return std::isfinite(v) || fail(std::string(name) + " is not a finite number");
    }
    bool whole(const std::string& name, int64_t fallback, int64_t lo, int64_t hi, int64_t& v) {
        double d = 0.0;
        if (!real(name.c_str(), static_cast<double>(fallback), d)) return false;
        if (d != std::floor(d) || d < static_cast<double>(lo) || d > static_cast<double>(hi)) {
            return fail(name + " must be a whole number of " + std::to_string(lo) + " .. " + std::to_string(hi));
        }
        v = static_cast<int64_t>(d);
        return true;
    }

    /// Operand `slot` as rows of `heads` heads of `dim` elements, columns
    /// [<slot>_at, ..) of its buffer's rows.
    bool heads(int slot, int64_t heads, int64_t dim, Dtype want, Operand& o) {
        if (!has(slot)) return fail(std::string("operand '") + kSlotNames[slot] + "' is missing");
        const KernelBuffer& b = km_.buffers[id(slot)];
        if (b.dtype != want) return fail(std::string("'") + kSlotNames[slot] + "' has another dtype than 'q'");
        o.buffer = id(slot);
        o.rows = b.dims[0];
        o.width = 1;
        for (size_t i = 1; i < b.dims.size(); ++i) o.width *= b.dims[i];
        if (o.rows > kMaxRows) return fail(std::string("'") + kSlotNames[slot] + "' has 2^31 rows or more");
        if (!whole(std::string(kSlotNames[slot]) + "_at", 0, 0, int64_t{1} << 40, o.at)) return false;
        if (o.at + heads * dim > o.width) {
            return fail(std::string("'") + kSlotNames[slot] + "' rows hold " + std::to_string(o.width) + " elements, columns " +
                        std::to_string(o.at) + " .. " + std::to_string(o.at + heads * dim) + " are needed");
        }
        return true;
    }

    /// Operand `slot` as a dense array of exactly `elements` (-1: any number).
    bool dense(int slot, Dtype want, int64_t elements, const char* type, Operand& o) {
        const KernelBuffer& b = km_.buffers[id(slot)];
        o.buffer = id(slot);
        o.rows = 1;
        for (const int64_t d : b.dims) o.rows *= d;
        o.width = o.rows;
        if (b.dtype != want) return fail(std::string("'") + kSlotNames[slot] + "' must be " + type);
        if (elements >= 0 && o.rows != elements) {
            return fail(std::string("'") + kSlotNames[slot] + "' must hold " + std::to_string(elements) + " elements");
        }
        return true;
    }

private:
    static bool rowsOfHeads(int s) {
        return s <= kOpPrefixV || s == kOpQOut || s == kOpKOut || s == kOpVOut || s == kOpOut;
    }
    const KernelModule& km_;
    const KernelNode& n_;
    std::string what_;
    std::string why_;
};

bool floatType(Dtype d) { return d == Dtype::F16 || d == Dtype::BF16 || d == Dtype::F32; }

/// heads, kv_heads, dim and q's dtype and rows, which the other operands go by.
bool shape(Reader& r, OperatorStep& o) {
    int64_t h = 0, g = 0, d = 0;
    if (!r.whole("heads", 0, 1, kMaxHeads, h) || !r.whole("kv_heads", h, 1, kMaxHeads, g) || !r.whole("dim", 0, 1, kMaxDim, d)) {
        return false;
    }
    if (h % g != 0) return r.fail("heads must be a multiple of kv_heads");
    if (!r.has(kOpQ)) return r.fail("operand 'q' is missing");
    if (!floatType(r.dtype(kOpQ))) return r.fail("'q' must be f16, bf16 or f32");
    o.heads = static_cast<int32_t>(h);
    o.kvHeads = static_cast<int32_t>(g);
    o.dim = static_cast<int32_t>(d);
    return r.heads(kOpQ, h, d, r.dtype(kOpQ), o.op[kOpQ]);
}

/// No output shares elements with another operand, but for outputs that take
/// the very place of their input (`inPlace`, slot pairs).
bool disjoint(Reader& r, const OperatorStep& o, const int64_t* columns, const std::vector<std::pair<int, int>>& inPlace) {
    for (int w = kFirstOpOutput; w < kOperandSlots; ++w) {
        if (o.op[w].buffer == kInvalidId) continue;
        for (int s = 0; s < kOperandSlots; ++s) {
            if (s == w || o.op[s].buffer != o.op[w].buffer) continue;
            if (o.op[w].at + columns[w] <= o.op[s].at || o.op[s].at + columns[s] <= o.op[w].at) continue;
            bool same = false;
            for (const auto& [in, out] : inPlace) same = same || (in == s && out == w && o.op[in].at == o.op[out].at);
            if (!same) {
                return r.fail(std::string("'") + kSlotNames[w] + "' overlaps '" + kSlotNames[s] + "'");
            }
        }
    }
    return true;
}

/// q_offsets holds the first row of each sequence and the end of the last.
bool sequences(Reader& r, OperatorStep& o) {
    if (!r.dense(kOpQOffsets, Dtype::I32, -1, "i32", o.op[kOpQOffsets])) return false;
    const int64_t n = o.op[kOpQOffsets].rows - 1;
    if (n < 1 || n > (1 << 20)) return r.fail("'q_offsets' must hold 2 .. 2^20 + 1 elements");
    o.sequences = static_cast<int32_t>(n);
    return true;
}

bool normRope(Reader& r, OperatorStep& o) {
    if (!r.names({kOpQ, kOpK, kOpV, kOpQWeight, kOpKWeight, kOpPositions, kOpSlots, kOpQOffsets, kOpQOut, kOpKOut, kOpVOut},
                 {"heads", "kv_heads", "dim", "eps", "theta", "rot", "interleaved", "section_0", "section_1", "section_2"}) ||
        !shape(r, o)) {
        return false;
    }
    const Dtype dt = r.dtype(kOpQ);
    const int64_t h = o.heads, g = o.kvHeads, d = o.dim, rows = o.op[kOpQ].rows;
    if (!r.heads(kOpK, g, d, dt, o.op[kOpK]) || !r.heads(kOpQOut, h, d, dt, o.op[kOpQOut]) ||
        !r.heads(kOpKOut, g, d, dt, o.op[kOpKOut])) {
        return false;
    }
    if (r.has(kOpV) != r.has(kOpVOut)) return r.fail("'v' and 'v_out' come together");
    if (r.has(kOpV) && (!r.heads(kOpV, g, d, dt, o.op[kOpV]) || !r.heads(kOpVOut, g, d, dt, o.op[kOpVOut]))) return false;
    if (o.op[kOpK].rows != rows || o.op[kOpQOut].rows != rows || (r.has(kOpV) && o.op[kOpV].rows != rows)) {
        return r.fail("'q', 'k', 'v' and 'q_out' must have the same rows");
    }
    if (r.has(kOpV) && o.op[kOpVOut].rows != o.op[kOpKOut].rows) return r.fail("'k_out' and 'v_out' must have the same rows");
    if (r.has(kOpSlots)) {
        if (!r.dense(kOpSlots, Dtype::I32, rows, "i32", o.op[kOpSlots])) return false;
    } else if (o.op[kOpKOut].rows != rows) {
        return r.fail("'k_out' must have the rows of 'k' where there are no slots");
    }
    if (r.has(kOpQWeight) != r.has(kOpKWeight)) return r.fail("'q_weight' and 'k_weight' come together");
    if (r.has(kOpQWeight)) {
        const Dtype wt = r.dtype(kOpQWeight);
        if (wt != dt && wt != Dtype::F32) return r.fail("weights must be f32 or of the dtype of 'q'");
        if (!r.dense(kOpQWeight, wt, d, "of one dtype", o.op[kOpQWeight]) ||
            !r.dense(kOpKWeight, wt, d, "of the dtype of 'q_weight'", o.op[kOpKWeight])) {
            return false;
        }
    }
    int64_t rot = 0, inter = 0;
    double theta = 0.0;
    if (!r.real("eps", 1e-6, o.eps) || !r.real("theta", 10000.0, theta) || !r.whole("rot", d, 0, d, rot) ||
        !r.whole("interleaved", 0, 0, 1, inter)) {
        return false;
    }
    if (o.eps < 0.0 || o.eps > 1.0) return r.fail("eps must be of 0 .. 1");
    if (!(theta >= 1.0 && theta <= 1e12)) return r.fail("theta must be of 1 .. 1e12");
    if (!r.has(kOpPositions)) rot = 0;
    if (rot % 2 != 0) return r.fail("rot must be even");
    o.rot = static_cast<int32_t>(rot);
    o.interleaved = inter != 0;
    for (int k = 0; k < 7 && rot > 0; ++k) o.power[k] = std::pow(theta, -2.0 * (1 << k) / static_cast<double>(rot));
    int64_t section[3] = {0, 0, 0};
    if (!r.whole("section_0", rot / 2, 0, kMaxDim, section[0]) || !r.whole("section_1", 0, 0, kMaxDim, section[1]) ||
        !r.whole("section_2", 0, 0, kMaxDim, section[2])) {
        return false;
    }
    if (r.has(kOpPositions)) {
        if (section[0] + section[1] + section[2] != rot / 2) return r.fail("the sections must add up to rot / 2");
        o.axes = section[2] > 0 ? 3 : section[1] > 0 ? 2 : 1;
        for (int i = 0; i < 3; ++i) o.sections[i] = static_cast<int32_t>(section[i]);
        if (!r.dense(kOpPositions, Dtype::I32, o.axes * rows, "i32", o.op[kOpPositions])) return false;
    }
    if (r.has(kOpQOffsets) && !sequences(r, o)) return false;
    int64_t columns[kOperandSlots];
    for (int s = 0; s < kOperandSlots; ++s) columns[s] = s == kOpQ || s == kOpQOut ? h * d : s >= kOpQWeight && s < kOpQOut ? o.op[s].width : g * d;
    std::vector<std::pair<int, int>> inPlace = {{kOpQ, kOpQOut}};
    if (!r.has(kOpSlots)) {
        inPlace.emplace_back(kOpK, kOpKOut);
        inPlace.emplace_back(kOpV, kOpVOut);
    }
    return disjoint(r, o, columns, inPlace);
}

bool attention(Reader& r, OperatorStep& o, bool prefix) {
    bool ok = prefix ? r.names({kOpQ, kOpK, kOpV, kOpPrefixK, kOpPrefixV, kOpPrefixLen, kOpQOffsets, kOpKvStart, kOpKvLen, kOpOut, kOpLse},
                               {"heads", "kv_heads", "dim", "scale", "causal"})
                     : r.names({kOpQ, kOpK, kOpV, kOpQOffsets, kOpKvStart, kOpKvLen, kOpOut, kOpLse},
                               {"heads", "kv_heads", "dim", "scale", "causal"});
    if (!ok || !shape(r, o)) return false;
    const Dtype dt = r.dtype(kOpQ);
    const int64_t h = o.heads, g = o.kvHeads, d = o.dim, rows = o.op[kOpQ].rows;
    if (!r.heads(kOpK, g, d, dt, o.op[kOpK]) || !r.heads(kOpV, g, d, dt, o.op[kOpV]) || !r.heads(kOpOut, h, d, dt, o.op[kOpOut])) {
        return false;
    }
    if (o.op[kOpOut].rows != rows) return r.fail("'q' and 'out' must have the same rows");
    if (o.op[kOpV].rows != o.op[kOpK].rows) return r.fail("'k' and 'v' must have the same rows");
    if (!r.has(kOpQOffsets)) return r.fail("operand 'q_offsets' is missing");
    if (!sequences(r, o)) return false;
    if (r.has(kOpKvStart) != r.has(kOpKvLen)) return r.fail("'kv_start' and 'kv_len' come together");
    if (r.has(kOpKvStart)) {
        if (!r.dense(kOpKvStart, Dtype::I32, o.sequences, "i32", o.op[kOpKvStart]) ||
            !r.dense(kOpKvLen, Dtype::I32, o.sequences, "i32", o.op[kOpKvLen])) {
            return false;
        }
    } else if (o.op[kOpK].rows != rows) {
        return r.fail("'k' must have the rows of 'q' where there is no 'kv_start'");
    }
    if (prefix) {
        if (!r.heads(kOpPrefixK, g, d, dt, o.op[kOpPrefixK]) || !r.heads(kOpPrefixV, g, d, dt, o.op[kOpPrefixV])) return false;
        if (o.op[kOpPrefixV].rows != o.op[kOpPrefixK].rows) return r.fail("'prefix_k' and 'prefix_v' must have the same rows");
        if (r.has(kOpPrefixLen) && !r.dense(kOpPrefixLen, Dtype::I32, 1, "i32", o.op[kOpPrefixLen])) return false;
    }
    if (r.has(kOpLse) && !r.dense(kOpLse, Dtype::F32, rows * h, "f32", o.op[kOpLse])) return false;
    int64_t causal = 0;
    if (!r.real("scale", 1.0 / std::sqrt(static_cast<double>(d)), o.scale) || !r.whole("causal", 1, 0, 1, causal)) return false;
    if (!(std::fabs(o.scale) >= 1e-20 && std::fabs(o.scale) <= 1e20)) return r.fail("scale must be of 1e-20 .. 1e20 in size");
    o.causal = causal != 0;
    int64_t columns[kOperandSlots];
    for (int s = 0; s < kOperandSlots; ++s) {
        columns[s] = s == kOpQ || s == kOpOut ? h * d : s <= kOpPrefixV ? g * d : o.op[s].width;
    }
    return disjoint(r, o, columns, {});
}

void* place(const Step& st, int slot, const std::vector<void*>& ptr, int bytes) {
    const Operand& o = st.oper.op[slot];
    if (o.buffer == kInvalidId) return nullptr;
    return static_cast<char*>(ptr[o.buffer]) + o.at * bytes;
}

}  // namespace

bool isOperator(const Step& st) { return st.kind == StepKind::NormRope || st.kind == StepKind::Attention; }

Result<Step> operatorStep(const KernelModule& km, const KernelNode& call) {
    Step st;
    Reader r(km, call);
    bool ok = false;
    if (call.math == MathOp::QkNormRope) {
        st.kind = StepKind::NormRope;
        st.what = "qk-norm-rope";
        ok = normRope(r, st.oper);
    } else {
        const bool prefix = call.math == MathOp::SharedPrefixAttention;
        st.kind = StepKind::Attention;
        st.what = prefix ? "shared-prefix-attention" : "attention";
        ok = attention(r, st.oper, prefix);
    }
    if (!ok) return err(ErrorCode::InvalidArgument, r.why());
    return st;
}

void fillNormRope(const KernelModule& km, const Step& st, const std::vector<void*>& ptr, mlkd_norm_rope& p) {
    p = {};
    const OperatorStep& o = st.oper;
    const Dtype dt = km.buffers[o.op[kOpQ].buffer].dtype;
    const int e = dtypeBytes(dt);
    p.q = place(st, kOpQ, ptr, e);
    p.k = place(st, kOpK, ptr, e);
    p.v = place(st, kOpV, ptr, e);
    p.q_out = place(st, kOpQOut, ptr, e);
    p.k_out = place(st, kOpKOut, ptr, e);
    p.v_out = place(st, kOpVOut, ptr, e);
    p.q_weight = place(st, kOpQWeight, ptr, 0);
    p.k_weight = place(st, kOpKWeight, ptr, 0);
    p.positions = static_cast<const int32_t*>(place(st, kOpPositions, ptr, 0));
    p.slots = static_cast<const int32_t*>(place(st, kOpSlots, ptr, 0));
    p.q_offsets = static_cast<const int32_t*>(place(st, kOpQOffsets, ptr, 0));
    p.dtype = operandCode(dt);
    p.weight_dtype = p.q_weight != nullptr ? operandCode(km.buffers[o.op[kOpQWeight].buffer].dtype) : p.dtype;
    p.heads = o.heads;
    p.kv_heads = o.kvHeads;
    p.dim = o.dim;
    p.rot = o.rot;
    p.interleaved = o.interleaved ? 1 : 0;
    p.axes = o.axes;
    p.sequences = o.sequences;
    for (int i = 0, end = 0; i < 3; ++i) p.section_end[i] = end += o.sections[i];
    p.tokens = o.op[kOpQ].rows;
    p.out_rows = o.op[kOpKOut].rows;
    p.q_stride = o.op[kOpQ].width;
    p.k_stride = o.op[kOpK].width;
    p.v_stride = o.op[kOpV].width;
    p.q_out_stride = o.op[kOpQOut].width;
    p.k_out_stride = o.op[kOpKOut].width;
    p.v_out_stride = o.op[kOpVOut].width;
    p.eps = o.eps;
    for (int k = 0; k < 7; ++k) p.power[k] = o.power[k];
}

void fillAttention(const KernelModule& km, const Step& st, const std::vector<void*>& ptr, mlkd_attention& p) {
    p = {};
    const OperatorStep& o = st.oper;
    const Dtype dt = km.buffers[o.op[kOpQ].buffer].dtype;
    const int e = dtypeBytes(dt);
    p.q = place(st, kOpQ, ptr, e);
    p.k = place(st, kOpK, ptr, e);
    p.v = place(st, kOpV, ptr, e);
    p.prefix_k = place(st, kOpPrefixK, ptr, e);
    p.prefix_v = place(st, kOpPrefixV, ptr, e);
    p.out = place(st, kOpOut, ptr, e);
    p.lse = static_cast<float*>(place(st, kOpLse, ptr, 0));
    p.q_offsets = static_cast<const int32_t*>(place(st, kOpQOffsets, ptr, 0));
    p.kv_start = static_cast<const int32_t*>(place(st, kOpKvStart, ptr, 0));
    p.kv_len = static_cast<const int32_t*>(place(st, kOpKvLen, ptr, 0));
    p.prefix_len = static_cast<const int32_t*>(place(st, kOpPrefixLen, ptr, 0));
    p.dtype = operandCode(dt);
    p.causal = o.causal ? 1 : 0;
    p.heads = o.heads;
    p.kv_heads = o.kvHeads;
    p.dim = o.dim;
    p.sequences = o.sequences;
    p.q_rows = o.op[kOpQ].rows;
    p.kv_rows = o.op[kOpK].rows;
    p.prefix_rows = o.op[kOpPrefixK].rows;
    p.q_stride = o.op[kOpQ].width;
    p.k_stride = o.op[kOpK].width;
    p.v_stride = o.op[kOpV].width;
    p.prefix_k_stride = o.op[kOpPrefixK].width;
    p.prefix_v_stride = o.op[kOpPrefixV].width;
    p.out_stride = o.op[kOpOut].width;
    p.scale = o.scale;
}

}  // namespace mlk::hip
