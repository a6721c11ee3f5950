// The training operators through include/vector_hip.hpp, on values that can be checked by hand.  --host: the
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
    ~Buffer() { vhip_free(0, p); }
    std::vector<float> read(size_t n) const {
        std::vector<float> v(n);
        detail::check(vhip_memcpy_dtoh(0, v.data(), p, n * sizeof(float)));  // after all work of the default stream
        return v;
    }
    float *f() const { return static_cast<float *>(p); }
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
    check("layer_norm refuses a null input", refused([&] {
              tr::layer_norm(at, DType::F32, DType::F32, {nullptr, 2, 4, 4}, nullptr, nullptr, 1e-5f, {}, nullptr, nullptr);
          }));
    check("softmax_xent refuses rows of another width", refused([&] {
              tr::softmax_xent(at, DType::F32, {&at, 2, 4, 4}, {&at, 3, 5, 5}, nullptr, nullptr, 1.f, nullptr, nullptr);
          }));
    check("orthogonalize refuses no steps", refused([&] {
              tr::NewtonSchulz ns;
              ns.steps = 0;
              tr::orthogonalize(at, DType::F32, 1, {&at, 2, 2, 2}, ns, {&at, 2});
          }));
    check("workspaces", tr::softmax_xent_workspace(DType::BF16, {nullptr, 100, 64, 64}, {nullptr, 1000, 64, 64}, true) >
                            tr::softmax_xent_workspace(DType::BF16, {nullptr, 100, 64, 64}, {nullptr, 1000, 64, 64}, false));
}

static void gpu() {
    // layer norm of (1, 3) is (-1, 1) at eps 0; its gradient for dy = (1, 0) is zero
    Buffer x(std::vector<float>{1.f, 3.f}), y(8), mean(4), rstd(4), dy(std::vector<float>{1.f, 0.f}), dx(8), dw(8), db(8);
    tr::Place at;
    const tr::Rows rx{x.p, 1, 2, 2};
    tr::layer_norm(at, DType::F32, DType::F32, rx, nullptr, nullptr, 0.f, {y.p, 2}, mean.f(), rstd.f());
    auto v = y.read(2);
    check("layer_norm", near(v[0], -1) && near(v[1], 1) && near(mean.read(1)[0], 2) && near(rstd.read(1)[0], 1));
    Buffer w1(tr::layer_norm_backward_workspace(rx));
    at.workspace = w1.p;
    at.workspace_bytes = tr::layer_norm_backward_workspace(rx);
    tr::layer_norm_backward(at, DType::F32, DType::F32, {dy.p, 1, 2, 2}, rx, nullptr, mean.f(), rstd.f(), {dx.p, 2}, dw.p, db.p);
    v = dx.read(2);
    const auto g = dw.read(2), b = db.read(2);
    check("layer_norm_backward", near(v[0], 0) && near(v[1], 0) && near(g[0], -1) && near(g[1], 0) && near(b[0], 1) && near(b[1], 0));

    // logits (ln 3, 0): p = (3/4, 1/4); target 0
    Buffer h(std::vector<float>{1.f}), table(std::vector<float>{std::log(3.f), 0.f}), target(std::vector<int64_t>{0}), loss(4), lse(4),
        dh(4), dt(8);
    const tr::Rows rh{h.p, 1, 1, 1}, rt{table.p, 2, 1, 1};
    const size_t need = tr::softmax_xent_workspace(DType::F32, rh, rt, true);
    Buffer w2(need);
    at.workspace = w2.p;
    at.workspace_bytes = need;
    const int64_t *ty = static_cast<const int64_t *>(target.p);
    tr::softmax_xent_grad(at, DType::F32, rh, rt, ty, nullptr, nullptr, 1.f, loss.f(), lse.f(), {dh.p, 1}, {dt.p, 1});
    const auto t = dt.read(2);
    check("softmax_xent_grad", near(loss.read(1)[0], std::log(4.0 / 3)) && near(lse.read(1)[0], std::log(4.0)) &&
                                   near(dh.read(1)[0], -0.25 * std::log(3.0)) && near(t[0], -0.25) && near(t[1], 0.25));
    tr::softmax_xent(at, DType::F32, rh, rt, ty, nullptr, 1.f, loss.f(), lse.f());
    check("softmax_xent", near(loss.read(1)[0], std::log(4.0 / 3)));

    // diag(3, 4) / 5 has singular values 0.6 and 0.8; one step of x -> a x + b x^3 + c x^5
    Buffer m(std::vector<float>{3.f, 0.f, 0.f, 4.f}), o(16);
    const size_t bytes = tr::orthogonalize_workspace(1, 2, 2);
    Buffer w3(bytes);
    at.workspace = w3.p;
    at.workspace_bytes = bytes;
    tr::NewtonSchulz ns;
    ns.steps = 1;
    tr::orthogonalize(at, DType::F32, 1, {m.p, 2, 2, 2}, ns, {o.p, 2});
    auto step = [&](double s) { return ns.a * s + ns.b * s * s * s + ns.c * std::pow(s, 5); };
    v = o.read(4);
    check("orthogonalize", near(v[0], step(0.6)) && near(v[3], step(0.8)) && near(v[1], 0) && near(v[2], 0));
}

int main(int argc, char **argv) {
    host();
    if (!(argc > 1 && std::strcmp(argv[1], "--host") == 0)) gpu();
    return failures ? 1 : 0;
}
