// LayerNormalization, RotaryPositions and Attention<BackendMI355X> through the C++ layer, floats, against plain loops
// in double.  Errors are compared with 1e-5 of the results' root mean square: sums of at most a hundred terms in 32 bits, 100 * 2^-24 = 6e-6.
#include "test_common.hpp"

#include <algorithm>

static std::vector<float> randn(size_t n, unsigned seed)
{
    std::mt19937 gen(seed);
    std::normal_distribution<float> d;
    std::vector<float> v(n);
    for (auto& x : v)
        x = d(gen);
    return v;
}

template <typename T>
struct Buffer
{
    explicit Buffer(const std::vector<T>& h) : Buffer(h.size())
    {
        DISTCONV_CHECK_HIP(hipMemcpy(p, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice));
    }
    explicit Buffer(size_t n) : n(n) { DISTCONV_CHECK_HIP(hipMalloc(&p, n * sizeof(T))); }
    ~Buffer() { (void) hipFree(p); }
    std::vector<T> host() const
    {
        std::vector<T> h(n);
        DISTCONV_CHECK_HIP(hipDeviceSynchronize());
        DISTCONV_CHECK_HIP(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
    T* p = nullptr;
    size_t n;
};

static bool close(const char* what, const std::vector<float>& got, const std::vector<double>& want)
{
    CHECK(got.size() == want.size());
    double error = 0, size = 0;
    for (size_t i = 0; i < got.size(); ++i)
    {
        error += (got[i] - want[i]) * (got[i] - want[i]);
        size += want[i] * want[i];
    }
    const bool ok = error <= 1e-10 * size;
    std::printf("%s: relative error %.2g %s\n", what, std::sqrt(error / size), ok ? "ok" : "FAILED");
    return ok;
}

// A haloed tensor whose channel is innermost: 20 channels, 6 x 4 cells, 3 samples.
static int test_norm()
{
    const Shape shape({20, 12, 4, 3});
    const Distribution dist = Distribution::make_overlapped_distribution(Shape({1, 2, 1, 1}), IntVector({0, 1, 0, 0}));
    const LocaleVirtual loc(0, 2);
    DevTensor<float> x(shape, loc, dist), y(shape, loc, dist), dy(shape, loc, dist), dx(shape, loc, dist);
    for (auto* t : {&x, &y, &dy, &dx})
        t->allocate();
    const size_t size = x.get_local_real_size(), rows = x.get_local_size() / 20;
    CHECK(size > static_cast<size_t>(x.get_local_size())); // there is a halo
    const auto hx = randn(size, 1), hdy = randn(size, 2), w = randn(20, 3), b = randn(20, 4);
    to_device(x, hx);
    to_device(dy, hdy);
    to_device(y, std::vector<float>(size, 7.0f));
    to_device(dx, std::vector<float>(size, 7.0f));
    Buffer<float> dw(w), db(b), scale(w), bias(b), mean(rows), rstd(rows);
    BackendMI355X backend;
    LayerNormalization<BackendMI355X> layer(backend, 1e-4);
    layer.forward(x, scale.p, bias.p, y, mean.p, rstd.p);
    layer.backward(x, dy, mean.p, rstd.p, scale.p, dx, dw.p, db.p);
    std::vector<double> wy(size, 7.0), wdx(size, 7.0), wdw(20), wdb(20);
    for (size_t r = 0; r < rows; ++r)
    {
        // cells in order, innermost first, as the local shape counts them
        const Shape& ls = x.get_local_shape();
        const size_t at = x.get_local_offset(ls.get_index(r * 20));
        double m = 0, v = 0, sum = 0, dot = 0;
        for (int c = 0; c < 20; ++c)
            m += hx[at + c] / 20.0;
        for (int c = 0; c < 20; ++c)
            v += (hx[at + c] - m) * (hx[at + c] - m) / 20.0;
        const double s = 1 / std::sqrt(v + 1e-4);
        for (int c = 0; c < 20; ++c)
        {
            const double h = (hx[at + c] - m) * s, g = static_cast<double>(hdy[at + c]) * w[c];
            wy[at + c] = h * w[c] + b[c];
            wdw[c] += hdy[at + c] * h;
            wdb[c] += hdy[at + c];
            sum += g / 20;
            dot += g * h / 20;
        }
        for (int c = 0; c < 20; ++c)
            wdx[at + c] = s * (static_cast<double>(hdy[at + c]) * w[c] - sum - (hx[at + c] - m) * s * dot);
    }
    int errors = 0;
    errors += !close("layer normalisation", to_host(y), wy);
    errors += !close("  gradient of the input", to_host(dx), wdx);
    errors += !close("  of the scale", dw.host(), wdw);
    errors += !close("  of the bias", db.host(), wdb);
    return errors;
}

static int test_rotary()
{
    const int tokens = 30, heads = 3, dim = 16;
    const std::vector<int> pairs = {3, 4};
    const auto hx = randn(tokens * heads * dim, 5);
    std::vector<int32_t> hp(2 * tokens);
    for (int i = 0; i < 2 * tokens; ++i)
        hp[i] = 37 * i - 400;
    Buffer<float> x(hx), y(hx.size());
    Buffer<int32_t> positions(hp);
    BackendMI355X backend;
    RotaryPositions<BackendMI355X> layer(backend, pairs);
    h2x_rotary r = {};
    r.dtype = H2X_F32;
    r.head_dim = dim;
    r.heads = heads;
    r.samples = 1;
    r.tokens = tokens;
    r.positions_axis_stride = tokens;
    r.x = r.y = {0, heads * dim, dim};
    layer.forward(r, x.p, positions.p, y.p);
    std::vector<double> want(hx.begin(), hx.end());
    for (int t = 0; t < tokens; ++t)
        for (int h = 0; h < heads; ++h)
            for (int i = 0; i < 7; ++i)
            {
                const double angle = hp[(i < 3 ? 0 : tokens) + t] * std::pow(10000.0, i < 3 ? -i / 3.0 : -(i - 3) / 4.0);
                double *u = &want[(t * heads + h) * dim + i], *v = u + 7;
                const double a = *u, b = *v;
                *u = a * std::cos(angle) - b * std::sin(angle);
                *v = a * std::sin(angle) + b * std::cos(angle);
            }
    int errors = !close("rotary positions", y.host(), want);
    layer.backward(r, y.p, positions.p, y.p); // turned back, in place
    errors += !close("  and back", y.host(), std::vector<double>(hx.begin(), hx.end()));
    return errors;
}

// Causal, two query heads to a key head.
static int test_attention()
{
    const int n = 2, t = 40, heads = 4, key_heads = 2, dim = 24;
    const auto hq = randn(n * t * heads * dim, 6), hk = randn(n * t * key_heads * dim, 7), hv = randn(n * t * key_heads * dim, 8),
               hd = randn(n * t * heads * dim, 9);
    Buffer<float> q(hq), k(hk), v(hv), d_o(hd), o(hq.size()), dq(hq.size()), dk(hk.size()), dv(hv.size()), lse(n * heads * t);
    h2x_attention a = {};
    a.dtype = H2X_F32;
    a.head_dim = dim;
    a.samples = n;
    a.query_heads = heads;
    a.key_heads = key_heads;
    a.queries = a.keys = t;
    a.window_left = -1;
    a.scale = 0.2;
    a.q = a.o = a.d_o = a.dq = {t * heads * dim, heads * dim, dim};
    a.k = a.v = a.dk = a.dv = {t * key_heads * dim, key_heads * dim, dim};
    BackendMI355X backend;
    Attention<BackendMI355X> layer(backend);
    layer.forward(a, q.p, k.p, v.p, o.p, lse.p);
    layer.backward(a, q.p, k.p, v.p, o.p, d_o.p, lse.p, dq.p, dk.p, dv.p);
    std::vector<double> wo(hq.size()), wq(hq.size()), wk(hk.size()), wv(hv.size());
    for (int b = 0; b < n; ++b)
        for (int h = 0; h < heads; ++h)
            for (int i = 0; i < t; ++i)
            {
                const size_t row = ((static_cast<size_t>(b) * t + i) * heads + h) * dim;
                const auto other = [&](int j) { return ((static_cast<size_t>(b) * t + j) * key_heads + h / 2) * dim; };
                std::vector<double> p(i + 1), dp(i + 1);
                double total = 0, delta = 0;
                for (int j = 0; j <= i; ++j)
                {
                    double s = 0;
                    for (int e = 0; e < dim; ++e)
                        s += static_cast<double>(hq[row + e]) * hk[other(j) + e];
                    total += p[j] = std::exp(0.2 * s);
                }
                for (int j = 0; j <= i; ++j)
                {
                    p[j] /= total;
                    for (int e = 0; e < dim; ++e)
                    {
                        wo[row + e] += p[j] * hv[other(j) + e];
                        dp[j] += static_cast<double>(hd[row + e]) * hv[other(j) + e];
                        wv[other(j) + e] += p[j] * hd[row + e];
                    }
                    delta += p[j] * dp[j];
                }
                for (int j = 0; j <= i; ++j)
                    for (int e = 0; e < dim; ++e)
                    {
                        const double ds = 0.2 * p[j] * (dp[j] - delta);
                        wq[row + e] += ds * hk[other(j) + e];
                        wk[other(j) + e] += ds * hq[row + e];
                    }
            }
    int errors = 0;
    errors += !close("attention", o.host(), wo);
    errors += !close("  gradient of the queries", dq.host(), wq);
    errors += !close("  of the keys", dk.host(), wk);
    errors += !close("  of the values", dv.host(), wv);
    return errors;
}

// A captured backward pass replays with the workspace that it was captured with, though larger calls of the layer followed.
static int test_graph()
{
    const int most = 160, heads = 2, dim = 8;
    const size_t size = most * heads * dim;
    const auto hq = randn(size, 10), hk = randn(size, 11), hv = randn(size, 12), hd = randn(size, 13);
    Buffer<float> q(hq), k(hk), v(hv), d_o(hd), o(size), dq(size), dk(size), dv(size), lse(heads * most);
    h2x_attention a = {};
    a.dtype = H2X_F32;
    a.head_dim = dim;
    a.samples = 1;
    a.query_heads = a.key_heads = heads;
    a.window_left = -1;
    a.scale = 0.3;
    a.q = a.o = a.d_o = a.dq = a.k = a.v = a.dk = a.dv = {0, heads * dim, dim};
    hipStream_t stream;
    DISTCONV_CHECK_HIP(hipStreamCreateWithFlags(&stream, hipStreamNonBlocking));
    DISTCONV_CHECK_HIP(hipDeviceSynchronize());
    int errors = 0;
    {
        BackendMI355X backend(stream);
        Attention<BackendMI355X> layer(backend);
        const auto run = [&](int tokens) {
            a.queries = a.keys = tokens;
            layer.forward(a, q.p, k.p, v.p, o.p, lse.p);
            layer.backward(a, q.p, k.p, v.p, o.p, d_o.p, lse.p, dq.p, dk.p, dv.p);
        };
        run(40);
        const auto want_q = dq.host(), want_k = dk.host(), want_v = dv.host();
        hipGraph_t graph;
        hipGraphExec_t replay;
        DISTCONV_CHECK_HIP(hipStreamBeginCapture(stream, hipStreamCaptureModeThreadLocal));
        run(40);
        DISTCONV_CHECK_HIP(hipStreamEndCapture(stream, &graph));
        DISTCONV_CHECK_HIP(hipGraphInstantiate(&replay, graph, nullptr, nullptr, 0));
        for (int i = 0; i < 3; ++i)
        {
            run(most); // (the first one needs a larger workspace)
            DISTCONV_CHECK_HIP(hipGraphLaunch(replay, stream));
            DISTCONV_CHECK_HIP(hipStreamSynchronize(stream));
            const auto same = [&](const Buffer<float>& b, const std::vector<float>& want) {
                const auto got = b.host();
                return std::equal(got.begin(), got.begin() + 40 * heads * dim, want.begin());
            };
            errors += !(same(dq, want_q) && same(dk, want_k) && same(dv, want_v));
        }
        DISTCONV_CHECK_HIP(hipGraphExecDestroy(replay));
        DISTCONV_CHECK_HIP(hipGraphDestroy(graph));
    }
    DISTCONV_CHECK_HIP(hipStreamDestroy(stream));
    std::printf("captured attention %s\n", errors ? "FAILED" : "ok");
    return errors;
}

int main()
{
    const int errors = test_norm() + test_rotary() + test_attention() + test_graph();
    std::printf(errors ? "test_tokens: %d FAILED\n" : "test_tokens: ok\n", errors);
    return finish(errors);
}
