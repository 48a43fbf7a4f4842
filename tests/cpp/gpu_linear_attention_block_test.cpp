// The operators of a linear-attention block through the sycldnn:: headers, in float
// and bfloat16, against sums in double: positions by rotation, the attention and a
// gated product, one behind another by events on two streams, and the gradients
// against differences.  With --host, what is refused without a GPU.
#include <portdnn/backend/hip_backend.h>
#include <portdnn/gated_matmul/launch.h>
#include <portdnn/linear_attention/launch.h>
#include <portdnn/rotary/launch.h>

#include <cmath>
#include <cstring>
#include <random>
#include <vector>

#include "check.h"

using namespace sycldnn;
using Backend = backend::HIPBackend;
using Doubles = std::vector<double>;

static float load(float v) { return v; }
static float load(bfloat16 v) {
  const unsigned bits = static_cast<unsigned>(v.bits) << 16;
  float f;
  std::memcpy(&f, &bits, 4);
  return f;
}
static void store(float v, float* to) { *to = v; }
static void store(float v, bfloat16* to) {
  unsigned bits;
  std::memcpy(&bits, &v, 4);
  to->bits = static_cast<std::uint16_t>((bits + 0x7FFF + (bits >> 16 & 1)) >> 16);
}

// n values of T on the device, and as doubles.
template <typename T>
struct Values {
  Doubles host;
  T* at;
  Backend* b;
  Values(Backend& be, size_t n, std::mt19937& gen, float size = 1.f) : b(&be) {
    std::normal_distribution<float> d(0.f, size);
    std::vector<T> raw(n);
    host.resize(n);
    for (size_t i = 0; i < n; ++i) {
      store(d(gen), &raw[i]);
      host[i] = load(raw[i]);
    }
    at = be.allocate<T>(n);
    (void)hipMemcpy(at, raw.data(), n * sizeof(T), hipMemcpyHostToDevice);
  }
  Values(Backend& be, size_t n) : host(n), at(be.allocate<T>(n)), b(&be) {
    (void)hipMemset(at, 0xff, n * sizeof(T));
  }
  Doubles read() const {
    std::vector<T> raw(host.size());
    (void)hipMemcpy(raw.data(), at, raw.size() * sizeof(T),
                    hipMemcpyDeviceToHost);
    Doubles v(raw.size());
    for (size_t i = 0; i < v.size(); ++i) v[i] = load(raw[i]);
    return v;
  }
  ~Values() { b->deallocate(at); }
};

// Some hundred fp32 operations and two roundings to the type (of a product of
// queries and keys, and of the output) on terms of up to ten times the result.
template <typename T>
static void check_all(const char* what, const Doubles& got, const Doubles& want) {
  const double rounding = std::is_same<T, float>::value ? 0x1p-24 : 0x1p-8;
  double scale = 0;
  for (double v : want) scale = std::max(scale, std::abs(v));
  size_t bad = 0;
  for (size_t i = 0; i < want.size(); ++i)
    if (!(std::abs(got[i] - want[i]) <=
          rounding * std::abs(want[i]) + (rounding + 6400 * 0x1p-24) * scale))
      ++bad;
  if (bad != 0)
    std::printf("%s: %zu of %zu values\n", what, bad, want.size());
  CHECK_EQ(bad, 0);
}

static const int batch = 2, steps = 130, heads = 4, groups = 2, keys = 24,
                 values = 40, rows = batch * steps, inner = heads * values,
                 hidden = 56;

static Doubles turn(const Doubles& x, const Doubles& table) {
  const int half = keys / 2;
  Doubles y(x.size());
  for (int r = 0; r < rows * groups; ++r)
    for (int i = 0; i < half; ++i) {
      const double w = 2 * M_PI * (r / groups % steps) * table[i];
      const double a = x[r * keys + i], b = x[r * keys + half + i];
      y[r * keys + i] = a * std::cos(w) - b * std::sin(w);
      y[r * keys + half + i] = a * std::sin(w) + b * std::cos(w);
    }
  return y;
}

static Doubles attend(const Doubles& q, const Doubles& k, const Doubles& v,
                      const Doubles& decay, Doubles* last = nullptr) {
  Doubles o(rows * inner);
  if (last != nullptr) last->clear();
  for (int b = 0; b < batch; ++b)
    for (int h = 0; h < heads; ++h) {
      Doubles s(keys * values);
      for (int t = 0; t < steps; ++t) {
        const int row = b * steps + t;
        const double* const kt = &k[(row * groups + h / 2) * keys];
        const double* const qt = &q[(row * groups + h / 2) * keys];
        for (int c = 0; c < values; ++c) {
          double sum = 0;
          for (int i = 0; i < keys; ++i) {
            double& at = s[i * values + c];
            at = std::exp(decay[h]) * at + kt[i] * v[(row * heads + h) * values + c];
            sum += qt[i] * at;
          }
          o[(row * heads + h) * values + c] = 0.2 * sum;
        }
      }
      if (last != nullptr) last->insert(last->end(), s.begin(), s.end());
    }
  return o;
}

template <typename T>
static void run_block() {
  std::mt19937 gen(5);
  hipStream_t streams[2];
  CHECK_EQ(hipStreamCreate(&streams[0]), hipSuccess);
  CHECK_EQ(hipStreamCreate(&streams[1]), hipSuccess);
  {
    Backend first(streams[0]), second(streams[1]);
    Values<T> q(first, rows * groups * keys, gen), k(first, rows * groups * keys, gen),
        v(first, rows * inner, gen);
    Values<float> decay(first, heads, gen, 0.f);
    std::vector<float> logs = {0.f, -0.01f, -0.1f, -1.f};
    (void)hipMemcpy(decay.at, logs.data(), sizeof(float) * heads,
                    hipMemcpyHostToDevice);
    decay.host.assign(logs.begin(), logs.end());
    Doubles table(keys / 2);
    CHECK(rotary::frequencies(keys, 10000.0, table.data()) == StatusCode::OK);
    double* const on_device = first.allocate<double>(table.size());
    (void)hipMemcpy(on_device, table.data(), sizeof(double) * table.size(),
                    hipMemcpyHostToDevice);

    // q and k turned, q in place
    rotary::Params tp{};
    tp.batch = batch;
    tp.steps = steps;
    tp.heads = groups;
    tp.channels = tp.turned = keys;
    tp.magnitude = 1.f;
    const Doubles turned_q = turn(q.host, table), turned_k = turn(k.host, table);
    Values<T> k2(first, rows * groups * keys);
    auto status = rotary::launch<T>(q.at, on_device, nullptr, q.at, tp, first);
    CHECK(status.status == StatusCode::OK);
    status = rotary::launch<T>(k.at, on_device, nullptr, k2.at, tp, first);
    CHECK(status.status == StatusCode::OK);

    // o, on the second stream
    linear_attention::Params ap{};
    ap.batch = batch;
    ap.steps = steps;
    ap.heads = heads;
    ap.key_heads = groups;
    ap.keys = keys;
    ap.values = values;
    ap.scale = 0.2f;
    const auto as = linear_attention::query_workspace_size<T>(ap);
    CHECK(as.required_size == 0);
    Values<T> aspace(second, as.recommended_size + 1), o(second, rows * inner);
    Values<float> last(second, batch * heads * keys * values);
    status = linear_attention::launch<T>(
        q.at, k2.at, v.at, decay.at, nullptr, nullptr, nullptr, o.at, last.at, ap,
        second, aspace.at, as.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);

    // m = gelu(o G) * (o U + c), on the first again
    Values<T> wg(first, inner * hidden, gen, 0.05f), wu(first, inner * hidden, gen, 0.05f),
        c(first, hidden, gen), m(first, rows * hidden), z(first, rows * hidden),
        u(first, rows * hidden);
    gated_matmul::Params gp{};
    gp.m = rows;
    gp.k = inner;
    gp.n = hidden;
    gp.activation = SNN_HIP_ACTIVATION_GELU;
    const auto gs = gated_matmul::query_workspace_size<T>(gp);
    Values<T> gspace(first, gs.recommended_size + 1);
    status = gated_matmul::launch<T>(o.at, wg.at, wu.at, nullptr, c.at, m.at, z.at,
                                     u.at, gp, first, gspace.at,
                                     gs.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);
    CHECK_EQ(hipStreamSynchronize(streams[0]), hipSuccess);

    const Doubles got_q = q.read(), got_k = k2.read(), got_o = o.read();
    check_all<T>("turned q", got_q, turned_q);
    check_all<T>("turned k", got_k, turned_k);
    Doubles want_last;
    check_all<T>("o", got_o, attend(got_q, got_k, v.host, decay.host, &want_last));
    check_all<float>("state", last.read(), want_last);
    Doubles want_m(rows * hidden), want_z(rows * hidden);
    for (int r = 0; r < rows; ++r)
      for (int n = 0; n < hidden; ++n) {
        double a = 0, b = c.host[n];
        for (int i = 0; i < inner; ++i) {
          a += got_o[r * inner + i] * wg.host[i * hidden + n];
          b += got_o[r * inner + i] * wu.host[i * hidden + n];
        }
        want_z[r * hidden + n] = a;
        want_m[r * hidden + n] = 0.5 * a * std::erfc(-a / std::sqrt(2.0)) * b;
      }
    check_all<T>("z", z.read(), want_z);
    check_all<T>("m", m.read(), want_m);

    // gradients: of the gated product along a direction of c, in which it is
    // linear, of the attention along one of v
    Values<T> dm(first, rows * hidden, gen), dc(first, hidden), dx(first, rows * inner);
    const auto ggs = gated_matmul::query_workspace_size<T>(gp, true);
    CHECK(ggs.required_size > 0);
    Values<T> ggspace(first, ggs.recommended_size);
    status = gated_matmul::launch_grad<T>(
        dm.at, o.at, wg.at, wu.at, z.at, u.at, dx.at, nullptr, nullptr, nullptr,
        dc.at, gp, first, ggspace.at, ggs.recommended_size);
    CHECK(status.status == StatusCode::OK);
    const auto ags = linear_attention::query_workspace_size<T>(ap, true);
    CHECK(ags.required_size > 0);
    Values<T> agspace(second, ags.recommended_size), do_(second, rows * inner, gen),
        dv(second, rows * inner), dq(second, rows * groups * keys);
    status = linear_attention::launch_grad<T>(
        do_.at, nullptr, q.at, k2.at, v.at, decay.at, nullptr, nullptr, nullptr,
        dq.at, nullptr, dv.at, nullptr, ap, second, agspace.at,
        ags.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);
    CHECK_EQ(hipStreamSynchronize(streams[1]), hipSuccess);
    const Doubles got_dc = dc.read(), got_z = z.read();
    Doubles want_dc(hidden);
    for (int r = 0; r < rows; ++r)
      for (int n = 0; n < hidden; ++n) {
        const double a = got_z[r * hidden + n];
        want_dc[n] += dm.host[r * hidden + n] * 0.5 * a *
                      std::erfc(-a / std::sqrt(2.0));
      }
    check_all<T>("dc", got_dc, want_dc);
    // (linear in v and in q: half the difference between two sides is exact)
    std::normal_distribution<double> d;
    auto along = [&](const Doubles& from, const Doubles& grad, bool of_v) {
      Doubles up = from, down = from;
      double moved = 0, size = 0;
      Doubles e(from.size());
      for (size_t i = 0; i < e.size(); ++i) {
        e[i] = d(gen);
        up[i] += e[i];
        down[i] -= e[i];
      }
      const Doubles a = of_v ? attend(got_q, got_k, up, decay.host)
                             : attend(up, got_k, v.host, decay.host);
      const Doubles b = of_v ? attend(got_q, got_k, down, decay.host)
                             : attend(down, got_k, v.host, decay.host);
      for (size_t i = 0; i < a.size(); ++i)
        moved += 0.5 * (a[i] - b[i]) * do_.host[i];
      double by = 0;
      for (size_t i = 0; i < e.size(); ++i) {
        by += e[i] * grad[i];
        size += std::abs(e[i] * grad[i]);
      }
      // (each gradient is off by two roundings of terms of up to ten times it)
      CHECK(std::abs(by - moved) <=
            (std::is_same<T, float>::value ? 1e-4 : 11 * 0x1p-8) * size);
    };
    along(v.host, dv.read(), true);
    along(got_q, dq.read(), false);
    first.deallocate(on_device);
  }
  (void)hipStreamDestroy(streams[0]);
  (void)hipStreamDestroy(streams[1]);
}

static void refusals() {
  Backend b;
  float* none = nullptr;
  bfloat16* nothing = nullptr;
  auto code = [](const SNNStatus& s) { return s.status; };
  gated_matmul::Params gp{};
  CHECK(code(gated_matmul::launch<float>(none, none, none, none, none, none, none,
                                         none, gp, b, none, 0)) ==
        StatusCode::InvalidParameter);
  CHECK(code(gated_matmul::launch_grad<bfloat16>(
            nothing, nothing, nothing, nothing, nothing, nothing, nothing, nothing,
            nothing, nothing, nothing, gp, b, nothing, 0)) ==
        StatusCode::InvalidParameter);
  rotary::Params tp{};
  CHECK(code(rotary::launch<float>(none, nullptr, nullptr, none, tp, b)) ==
        StatusCode::InvalidParameter);
  double table[4];
  CHECK(rotary::frequencies(8, 10000.0, table) == StatusCode::OK);
  CHECK(std::abs(table[0] * 2 * M_PI - 1) < 1e-15);
  CHECK(rotary::frequencies(7, 10000.0, table) == StatusCode::InvalidParameter);
  linear_attention::Params ap{};
  CHECK(code(linear_attention::launch<bfloat16>(
            nothing, nothing, nothing, none, nullptr, nullptr, none, nothing, none,
            ap, b, nothing, 0)) == StatusCode::InvalidParameter);
  CHECK(code(linear_attention::launch_grad<float>(
            none, none, none, none, none, none, nullptr, nullptr, none, none, none,
            none, none, ap, b, none, 0)) == StatusCode::InvalidParameter);
  // elements of the launch's type
  ap.batch = 1;
  ap.steps = 4096;
  ap.heads = ap.key_heads = 1;
  ap.keys = ap.values = 64;
  ap.scale = 1.f;
  CHECK(linear_attention::query_workspace_size<bfloat16>(ap).recommended_size > 0);
  CHECK(linear_attention::query_workspace_size<bfloat16>(ap).required_size == 0);
}

int main(int argc, char** argv) {
  refusals();
  if (argc < 2 || std::strcmp(argv[1], "--host") != 0) {
    run_block<float>();
    run_block<bfloat16>();
  }
  return report("linear_attention_block");
}
