// Attention, head norms and clipping through include/vector_hip.hpp, on values that can be checked by hand.  --host: the
// refusals alone, which need no GPU.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "vector_hip.hpp"

using namespace vector_hip;
namespace tr = vector_hip::training;

static int failures = 0;
static void check(const char *name, bool ok) {
    std::printf("%s %s\n", ok ? "PASS" : "FAIL", name);
    failures += !ok;
}

// Device memory that lives as long as the test.
struct Buffer {
    void *p = nullptr;
    explicit Buffer(size_t bytes) { detail::check(vhip_malloc(0, bytes, &p)); }
    template <class T>
    explicit Buffer(const std::vector<T> &v) : Buffer(v.size() * sizeof(T)) {
        detail::check(vhip_memcpy_htod(0, p, v.data(), v.size() * sizeof(T)));
    }
    Buffer(const Buffer &) = delete;
    Buffer &operator=(const Buffer &) = delete;
    ~Buffer() { vhip_free(0, p); }
    std::vector<float> read(size_t n) const {
        std::vector<float> v(n);
        detail::check(vhip_memcpy_dtoh(0, v.data(), p, n * sizeof(float)));  // after all work of the default stream
        return v;
    }
    float *f() const { return static_cast<float *>(p); }
    const int64_t *i() const { return static_cast<const int64_t *>(p); }
    vhip_heads heads(size_t token, size_t head) const { return {p, token, head}; }
};

static bool near(float a, double b, double tol = 1e-5) { return std::fabs(a - b) <= tol; }

template <class F>
static bool refused(F f) {
    try {
        f();
    } catch (const CudaError &e) {
        return e.kind() == CudaError::Kind::InvalidConfig;
    }
    return false;
}

static void host() {
    tr::Place at;
    int x = 0;
    const vhip_heads h{&x, 8, 4};
    check("attention refuses heads that are no multiple", refused([&] {
              tr::attention(at, DType::F32, {h, h, h, 2, 2, 3, 2, 4}, {1, (const int64_t *)&x, nullptr}, true, 1.f, h, nullptr);
          }));
    check("attention_backward refuses a null lse", refused([&] {
              tr::attention_backward(at, DType::F32, h, {h, h, h, 2, 2, 2, 2, 4}, h, nullptr, {1, (const int64_t *)&x, nullptr}, true, 1.f, h, h, h);
          }));
    check("qk_norm_rotary refuses an odd number of columns", refused([&] {
              tr::HeadNorm n;
              n.q = n.k = h;
              n.tokens = n.heads = n.kv_heads = 1;
              n.dim = 4;
              n.rotary = 3;
              tr::qk_norm_rotary(at, DType::F32, DType::F32, n, h, h);
          }));
    check("clip_gradients refuses an array twice", refused([&] {
              tr::clip_gradients(at, {{&x, &x, 1, VHIP_DTYPE_F32, VHIP_DTYPE_F32}, {&x, &x, 1, VHIP_DTYPE_F32, VHIP_DTYPE_F32}}, 1.f, 0.f, nullptr);
          }));
}

static void gpu() {
    // one head of one column: q = (1, 1), k = (ln 3, 0), v = (4, 8); causal: the first row sees key 0 alone, the
    // second has weights (3/4, 1/4)
    const float ln3 = std::log(3.f);
    Buffer q(std::vector<float>{1.f, 1.f}), k(std::vector<float>{ln3, 0.f}), v(std::vector<float>{4.f, 8.f}), offsets(std::vector<int64_t>{0, 2});
    Buffer out(64), lse(64), dout(std::vector<float>{0.f, 1.f}), dq(64), dk(64), dv(64);
    tr::Attended x{q.heads(1, 1), k.heads(1, 1), v.heads(1, 1), 2, 2, 1, 1, 1};
    const tr::Sequences s{1, offsets.i(), nullptr};
    Buffer w(tr::attention_workspace(DType::F32, x, s) + 16), w2(tr::attention_backward_workspace(DType::F32, x, s));
    tr::Place at;
    at.workspace = w.p;
    at.workspace_bytes = tr::attention_workspace(DType::F32, x, s);
    tr::attention(at, DType::F32, x, s, true, 1.f, out.heads(1, 1), lse.f());
    auto o = out.read(2), l = lse.read(2);
    check("attention", near(o[0], 4) && near(o[1], 5) && near(l[0], ln3) && near(l[1], std::log(4.0)));
    at.workspace = w2.p;
    at.workspace_bytes = tr::attention_backward_workspace(DType::F32, x, s);
    tr::attention_backward(at, DType::F32, dout.heads(1, 1), x, out.heads(1, 1), lse.f(), s, true, 1.f, dq.heads(1, 1), dk.heads(1, 1), dv.heads(1, 1));
    // ds = p (v - 5) = (-3/4, 3/4)
    const auto a = dq.read(2), b = dk.read(2), c = dv.read(2);
    check("attention_backward", near(a[0], 0) && near(a[1], -0.75 * ln3) && near(b[0], -0.75) && near(b[1], 0.75) && near(c[0], 0.75) && near(c[1], 0.25));

    // (3, 4) over its root mean square, turned by a quarter: (-4, 3) / sqrt(12.5); its own gradient is zero
    const double r = 1 / std::sqrt(12.5);
    Buffer hq(std::vector<float>{3.f, 4.f}), hk(std::vector<float>{1.f, 1.f}), pos(std::vector<int64_t>{1}), freq(std::vector<float>{1.5707964f}), qo(64), ko(64),
        gq(64), gk(64), gw(64), gv(64);
    tr::HeadNorm n;
    n.q = hq.heads(2, 2);
    n.k = hk.heads(2, 2);
    n.tokens = n.heads = n.kv_heads = 1;
    n.dim = n.rotary = 2;
    n.positions = pos.i();
    n.frequencies = freq.f();
    n.eps = 0.f;
    tr::qk_norm_rotary(at, DType::F32, DType::F32, n, qo.heads(2, 2), ko.heads(2, 2));
    const auto y = qo.read(2), z = ko.read(2);
    check("qk_norm_rotary", near(y[0], -4 * r) && near(y[1], 3 * r) && near(z[0], -1) && near(z[1], 1));
    Buffer w3(tr::qk_norm_rotary_backward_workspace(n));
    at.workspace = w3.p;
    at.workspace_bytes = tr::qk_norm_rotary_backward_workspace(n);
    tr::qk_norm_rotary_backward(at, DType::F32, DType::F32, qo.heads(2, 2), ko.heads(2, 2), n, gq.heads(2, 2), gk.heads(2, 2), gw.p, gv.p);
    const auto g = gq.read(2), t = gw.read(2), u = gv.read(2);
    check("qk_norm_rotary_backward", near(g[0], 0) && near(g[1], 0) && near(t[0], 9 * r * r) && near(t[1], 16 * r * r) && near(u[0], 1) && near(u[1], 1));

    // (3), (0, 4): norm 5, clipped to 1
    Buffer g1(std::vector<float>{3.f}), g2(std::vector<float>{0.f, 4.f}), o2(64), nrm(64), w4(tr::clip_gradients_workspace(2));
    at.workspace = w4.p;
    at.workspace_bytes = tr::clip_gradients_workspace(2);
    tr::gradient_norm(at, {{g1.p, nullptr, 1, VHIP_DTYPE_F32, VHIP_DTYPE_F32}, {g2.p, nullptr, 2, VHIP_DTYPE_F32, VHIP_DTYPE_F32}}, nrm.f());
    check("gradient_norm", near(nrm.read(1)[0], 5));
    tr::clip_gradients(at, {{g1.p, g1.p, 1, VHIP_DTYPE_F32, VHIP_DTYPE_F32}, {g2.p, o2.p, 2, VHIP_DTYPE_F32, VHIP_DTYPE_F32}}, 1.f, 0.f, nrm.f());
    check("clip_gradients", near(g1.read(1)[0], 0.6) && near(o2.read(2)[1], 0.8) && near(g2.read(2)[1], 4) && near(nrm.read(1)[0], 5));
}

int main(int argc, char **argv) {
    host();
    if (!(argc > 1 && std::strcmp(argv[1], "--host") == 0)) gpu();
    return failures ? 1 : 0;
}
