// Registries of part kinds: one name -> factory table for each role.
#include <mutex>

#include "../csrc/kernels.h"
#include "part.h"

namespace jb {

const char *step_kind_name(StepKind k) {
    return k == PREFILL ? "prefill" : k == DECODE ? "decode" : "extend";
}

namespace {
struct Tables {
    std::map<std::string, std::map<std::string, PartFactory>> parts;
    std::map<std::string, BlockFactory> blocks;
    std::mutex mu;
};
Tables &raw() {
    static Tables *t = new Tables();
    return *t;
}
Tables &ready() {
    static std::once_flag once;
    std::call_once(once, [] {
        register_builtin_norms();
        register_builtin_positions();
        register_builtin_mixers();
        register_builtin_feed_forwards();
        register_builtin_blocks();
        register_recurrent_mixers();
        register_routed_feed_forwards();
        register_pair_mixers();
    });
    return raw();
}
bool known_role(const std::string &r) {
    return r == "mixer" || r == "feed_forward" || r == "norm" || r == "position";
}
}  // namespace

void register_part(const std::string &role, const std::string &kind, PartFactory f) {
    if (!known_role(role)) fail(JB_LLM_EINVAL, "no role '" + role + "' (mixer, feed_forward, norm, position)");
    Tables &t = raw();
    std::lock_guard<std::mutex> lock(t.mu);
    t.parts[role][kind] = std::move(f);
}

void register_block(const std::string &kind, BlockFactory f) {
    Tables &t = raw();
    std::lock_guard<std::mutex> lock(t.mu);
    t.blocks[kind] = std::move(f);
}

std::vector<std::string> registered_parts(const std::string &role) {
    Tables &t = ready();
    std::lock_guard<std::mutex> lock(t.mu);
    std::vector<std::string> out;
    if (role == "block") {
        for (auto &kv : t.blocks) out.push_back(kv.first);
    } else {
        for (auto &kv : t.parts[role]) out.push_back(kv.first);
    }
    return out;
}

std::unique_ptr<Part> build_part(const std::string &role, const PartSpec &spec, DType dt, Device *dev) {
    if (!known_role(role)) fail(JB_LLM_EINVAL, "no role '" + role + "' (mixer, feed_forward, norm, position)");
    if (dt != F32 && dt != BF16) fail(JB_LLM_EINVAL, "the compute dtype is float32 or bfloat16");
    PartFactory f;
    {
        Tables &t = ready();
        std::lock_guard<std::mutex> lock(t.mu);
        auto &table = t.parts[role];
        auto it = table.find(spec.kind);
        if (it == table.end()) {
            std::string known;
            for (auto &kv : table) known += (known.empty() ? "" : ", ") + kv.first;
            config_error("no " + role + " of kind '" + spec.kind + "'; registered: " + known);
        }
        f = it->second;
    }
    return f(spec, dt, dev);
}

template <class T>
static std::unique_ptr<T> as_role(std::unique_ptr<Part> p, const char *role, const PartSpec &spec) {
    T *t = dynamic_cast<T *>(p.get());
    if (!t) config_error(std::string("the part registered as ") + role + " '" + spec.kind + "' is not a " + role);
    p.release();
    return std::unique_ptr<T>(t);
}

std::unique_ptr<Mixer> build_mixer(const PartSpec &s, DType dt, Device *d) {
    return as_role<Mixer>(build_part("mixer", s, dt, d), "mixer", s);
}
std::unique_ptr<FeedForward> build_feed_forward(const PartSpec &s, DType dt, Device *d) {
    return as_role<FeedForward>(build_part("feed_forward", s, dt, d), "feed_forward", s);
}
std::unique_ptr<Norm> build_norm(const PartSpec &s, DType dt, Device *d) {
    return as_role<Norm>(build_part("norm", s, dt, d), "norm", s);
}
std::unique_ptr<PositionEncoding> build_position(const PartSpec &s, DType dt, Device *d) {
    return as_role<PositionEncoding>(build_part("position", s, dt, d), "position", s);
}

std::unique_ptr<Block> build_block(const LayerSpec &ls, DType dt, Device *dev) {
    const std::string &kind = ls.block;
    BlockFactory bf;
    {
        Tables &t = ready();
        std::lock_guard<std::mutex> lock(t.mu);
        auto it = t.blocks.find(kind);
        if (it == t.blocks.end()) {
            std::string known;
            for (auto &kv : t.blocks) known += (known.empty() ? "" : ", ") + kv.first;
            config_error("no block arrangement '" + kind + "'; registered: " + known);
        }
        bf = it->second;
    }
    BlockParts p;
    p.mixer = build_mixer(ls.mixer, dt, dev);
    // an arrangement whose sublayers read the residual stream itself names no mixer_norm
    if (!ls.mixer_norm.kind.empty()) p.mixer_norm = build_norm(ls.mixer_norm, dt, dev);
    if (!ls.feed_forward.kind.empty()) {
        p.feed_forward = build_feed_forward(ls.feed_forward, dt, dev);
        // an arrangement whose sublayers share one norm names no ffn_norm
        if (!ls.ffn_norm.kind.empty()) p.ffn_norm = build_norm(ls.ffn_norm, dt, dev);
    }
    if (!ls.post_mixer_norm.kind.empty()) p.post_mixer_norm = build_norm(ls.post_mixer_norm, dt, dev);
    if (!ls.post_ffn_norm.kind.empty() && p.feed_forward) p.post_ffn_norm = build_norm(ls.post_ffn_norm, dt, dev);
    return bf(std::move(p), ls, dt, dev);
}

DevTensor Part::take(TensorMap &t, const std::string &name) {
    auto it = t.find(name);
    if (it == t.end()) fail(JB_LLM_EOPEN, "tensor " + name + " is missing");
    DevTensor v = it->second;
    t.erase(it);
    return v;
}

DevTensor fuse_rows(Device &dev, std::vector<DevTensor> &mats) {
    if (mats.empty()) fail(JB_LLM_EINVAL, "fuse_rows: nothing to fuse");
    if (mats.size() == 1) return mats[0];
    DType dt = mats[0].dt;
    long long cols = mats[0].shape.at(1), rows = 0;
    for (auto &m : mats) {
        if (m.dt == F32) dt = F32;
        if (m.shape.size() != 2 || m.shape[1] != cols) fail(JB_LLM_EINVAL, "fuse_rows: rows of unequal length");
        rows += m.shape[0];
    }
    dev.make_current();
    DevTensor out = dev.tensor(dt, {rows, cols});
    size_t at = 0;
    for (auto &m : mats) {
        if (jb_convert(m.ptr, m.dt, (char *)out.ptr + at, dt, m.numel(), dev.stream) != 0)
            fail(JB_LLM_EFAIL, "fuse_rows: the copy could not be launched");
        at += (size_t)m.numel() * dtype_size(dt);
    }
    dev.sync();      // the sources are freed when the caller lets go of them
    for (auto &m : mats) m = DevTensor();
    return out;
}

int pack_matrix(Device &dev, DevTensor &w) {
    if (w.shape.size() != 2 || (w.dt != F32 && w.dt != BF16) || w.shape[0] > 0x7fffffff || w.shape[1] > 0x7fffffff)
        fail(JB_LLM_EINVAL, "pack_matrix: not a matrix of floats");
    dev.make_current();
    DevTensor out = dev.tensor(MX4, w.shape);
    const int rows = (int)w.shape[0], k = (int)w.shape[1];
    if (jb_mx4_quantize(w.ptr, w.dt, out.ptr, (char *)out.ptr + mx4_code_bytes(rows, k), rows, k, 0, dev.stream) != 0)
        fail(JB_LLM_EFAIL, "pack_matrix: the kernel could not be launched");
    dev.sync();      // the floats are freed when their last owner lets go of them
    w = out;
    return 1;
}

// Several matrices with equally many rows as one, columns one after the other (the down
// matrices of a routed feed-forward's experts: one product over all experts' values).
DevTensor fuse_cols(Device &dev, std::vector<DevTensor> &mats) {
    if (mats.empty()) fail(JB_LLM_EINVAL, "fuse_cols: nothing to fuse");
    if (mats.size() == 1) return mats[0];
    DType dt = mats[0].dt;
    long long rows = mats[0].shape.at(0), cols = 0;
    for (auto &m : mats) {
        if (m.dt == F32) dt = F32;
        if (m.shape.size() != 2 || m.shape[0] != rows) fail(JB_LLM_EINVAL, "fuse_cols: columns of unequal length");
        cols += m.shape[1];
    }
    dev.make_current();
    DevTensor out = dev.tensor(dt, {rows, cols});
    size_t es = dtype_size(dt), at = 0;
    for (auto &m : mats) {
        DevTensor src = m;
        if (m.dt != dt) {
            src = dev.tensor(dt, m.shape);
            if (jb_convert(m.ptr, m.dt, src.ptr, dt, m.numel(), dev.stream) != 0)
                fail(JB_LLM_EFAIL, "fuse_cols: the conversion could not be launched");
        }
        size_t w = (size_t)m.shape[1] * es;
        cuda_check(cudaMemcpy2DAsync((char *)out.ptr + at, (size_t)cols * es, src.ptr, w, w, (size_t)rows,
                                     cudaMemcpyDeviceToDevice, dev.stream), "fuse_cols: placing a matrix");
        dev.sync();
        at += w;
    }
    for (auto &m : mats) m = DevTensor();
    return out;
}

}  // namespace jb
