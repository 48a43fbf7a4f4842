// The operators for sequences through the sycldnn:: headers, in float and
// bfloat16, against sums in double: a product with its epilogue, a gated norm
// and a recurrence, one behind another by events on two streams, and their
// gradients against differences.  With --host, what is refused without a GPU.
#include <portdnn/backend/hip_backend.h>
#include <portdnn/linear_recurrence/launch.h>
#include <portdnn/matmul_bias_act/launch.h>
#include <portdnn/residual_norm/launch.h>

#include <cmath>
#include <cstring>
#include <random>
#include <vector>

#include "check.h"

using namespace sycldnn;
using Backend = backend::HIPBackend;

static float round_to(float v, float) { return v; }
static float round_to(float v, bfloat16) {
  unsigned bits;
  std::memcpy(&bits, &v, 4);
  bits += 0x7FFF + (bits >> 16 & 1);
  bits &= 0xFFFF0000u;
  std::memcpy(&v, &bits, 4);
  return v;
}
static void store(float v, float* to) { *to = v; }
static void store(float v, bfloat16* to) {
  unsigned bits;
  std::memcpy(&bits, &v, 4);
  to->bits = static_cast<std::uint16_t>(bits >> 16);
}
static float load(float v) { return v; }
static float load(bfloat16 v) {
  const unsigned bits = static_cast<unsigned>(v.bits) << 16;
  float f;
  std::memcpy(&f, &bits, 4);
  return f;
}

// n values of T on the device (that T can hold) and as doubles.
template <typename T>
struct Values {
  std::vector<double> host;
  T* at;
  Backend* b;
  Values(Backend& be, size_t n, std::mt19937& gen, float shift = 0.f) : b(&be) {
    std::normal_distribution<float> d(shift, 1.f);
    std::vector<T> raw(n);
    host.resize(n);
    for (size_t i = 0; i < n; ++i) {
      const float v = round_to(d(gen), T{});
      host[i] = v;
      store(v, &raw[i]);
    }
    at = be.allocate<T>(n);
    (void)hipMemcpy(at, raw.data(), n * sizeof(T), hipMemcpyHostToDevice);
  }
  Values(Backend& be, size_t n) : host(n), at(be.allocate<T>(n)), b(&be) {
    (void)hipMemset(at, 0xff, n * sizeof(T));
  }
  std::vector<double> read() const {
    std::vector<T> raw(host.size());
    (void)hipMemcpy(raw.data(), at, raw.size() * sizeof(T),
                    hipMemcpyDeviceToHost);
    std::vector<double> v(raw.size());
    for (size_t i = 0; i < v.size(); ++i) v[i] = load(raw[i]);
    return v;
  }
  ~Values() { b->deallocate(at); }
};

static double sig(double v) { return 1.0 / (1.0 + std::exp(-v)); }
// A few hundred fp32 operations on terms of up to ten times the result, and the
// rounding of an output.
template <typename T>
static bool near(double got, double want, double scale) {
  const double rounding = std::is_same<T, float>::value ? 0x1p-24 : 0x1p-8;
  return std::abs(got - want) <=
         rounding * std::abs(want) + 640 * 0x1p-24 * scale;
}
template <typename T>
static void check_all(const char* what, const std::vector<double>& got,
                      const std::vector<double>& want) {
  double scale = 0;
  for (double v : want) scale = std::max(scale, std::abs(v));
  size_t bad = 0;
  for (size_t i = 0; i < want.size(); ++i)
    if (!near<T>(got[i], want[i], scale)) ++bad;
  if (bad != 0)
    std::printf("%s: %zu of %zu values\n", what, bad, want.size());
  CHECK_EQ(bad, 0);
}

template <typename T>
static void run_block() {
  std::mt19937 gen(5);
  hipStream_t streams[2];
  CHECK_EQ(hipStreamCreate(&streams[0]), hipSuccess);
  CHECK_EQ(hipStreamCreate(&streams[1]), hipSuccess);
  {
    Backend first(streams[0]), second(streams[1]);
    const int batch = 2, steps = 130, width = 24, inner = 20;
    const int rows = batch * steps, n = 2 * inner;

    // (x, forget) = u W + bias
    Values<T> u(first, rows * width, gen), w(first, width * n, gen),
        bias(first, n, gen, 1.f), p(first, rows * n);
    matmul_bias_act::Params mp{};
    mp.m = rows;
    mp.k = width;
    mp.n = n;
    const auto ws = matmul_bias_act::query_workspace_size<T>(mp);
    CHECK(ws.required_size <= ws.recommended_size);
    Values<T> space(first, ws.recommended_size + 1);
    auto status = matmul_bias_act::launch<T>(
        u.at, w.at, bias.at, nullptr, p.at, nullptr, mp, first, space.at,
        ws.recommended_size);
    CHECK(status.status == StatusCode::OK);

    // h, on the second stream
    linear_recurrence::Params rp{};
    rp.batch = batch;
    rp.steps = steps;
    rp.channels = inner;
    rp.row_stride = n;
    rp.grad_row_stride = n;
    const auto rs = linear_recurrence::query_workspace_size<T>(rp);
    CHECK(rs.recommended_size > 0);
    Values<T> rspace(second, rs.recommended_size);
    Values<T> h(second, rows * inner);
    Values<float> last(second, batch * inner);
    status = linear_recurrence::launch<T>(
        p.at, p.at + inner, nullptr, nullptr, nullptr, nullptr, h.at, last.at,
        rp, second, rspace.at, rs.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);

    // y = rms(h) weight
    Values<T> weight(first, inner, gen, 1.f), y(first, rows * inner);
    residual_norm::Params np{};
    np.rows = rows;
    np.channels = inner;
    np.post_norm = SNN_HIP_NORM_RMS;
    np.epsilon = 1e-6f;
    Values<float> stats(first, rows * 4);
    residual_norm::Tensors t{};
    t.x = h.at;
    t.post_weight = weight.at;
    t.sum = y.at;
    t.stats = stats.at;
    status = residual_norm::launch<T>(t, np, first, {status.event});
    CHECK(status.status == StatusCode::OK);
    status.event.wait_and_throw();

    const std::vector<double> got_p = p.read(), got_h = h.read();
    std::vector<double> want_p(rows * n), want_h(rows * inner),
        want_y(rows * inner), want_last(batch * inner);
    for (int r = 0; r < rows; ++r)
      for (int j = 0; j < n; ++j) {
        double s = bias.host[j];
        for (int k = 0; k < width; ++k)
          s += u.host[r * width + k] * w.host[k * n + j];
        want_p[r * n + j] = s;
      }
    auto recur = [&](const std::vector<double>& from) {
      std::vector<double> out(rows * inner);
      for (int b = 0; b < batch; ++b)
        for (int c = 0; c < inner; ++c) {
          double s = 0;
          for (int step = 0; step < steps; ++step) {
            const double* at = &from[(b * steps + step) * n];
            const double a = sig(at[inner + c]);
            s = a * s + (1 - a) * at[c];
            out[(b * steps + step) * inner + c] = s;
          }
        }
      return out;
    };
    // (each against what the kernel before it wrote)
    want_h = recur(got_p);
    for (int i = 0; i < batch * inner; ++i)
      want_last[i] = want_h[((i / inner) * steps + steps - 1) * inner + i % inner];
    for (int r = 0; r < rows; ++r) {
      double s = 0;
      for (int c = 0; c < inner; ++c)
        s += got_h[r * inner + c] * got_h[r * inner + c];
      for (int c = 0; c < inner; ++c)
        want_y[r * inner + c] = got_h[r * inner + c] /
                                std::sqrt(s / inner + 1e-6) * weight.host[c];
    }
    check_all<T>("product", got_p, want_p);
    check_all<T>("recurrence", got_h, want_h);
    check_all<float>("state", last.read(), want_last);
    check_all<T>("norm", y.read(), want_y);

    // The gradient of sum(dy y) goes back through all three.
    Values<T> dy(first, rows * inner, gen), dh(first, rows * inner),
        dweight(first, inner), dp(first, rows * n), du(first, rows * width),
        dw(first, width * n), dbias(first, n);
    const auto ns = residual_norm::query_grad_workspace_size<T>(np);
    Values<T> nspace(first, ns.recommended_size + 1);
    residual_norm::Gradients g{};
    g.grad_sum = dy.at;
    g.grad_x = dh.at;
    g.grad_post_weight = dweight.at;
    status = residual_norm::launch_grad<T>(t, g, np, first, nspace.at,
                                           ns.recommended_size);
    CHECK(status.status == StatusCode::OK);
    status = linear_recurrence::launch_grad<T>(
        dh.at, nullptr, p.at, p.at + inner, nullptr, nullptr, nullptr, nullptr,
        h.at, dp.at, dp.at + inner, nullptr, nullptr, rp, second, rspace.at,
        rs.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);
    const auto gs = matmul_bias_act::query_workspace_size<T>(mp, true);
    Values<T> gspace(first, gs.recommended_size + 1);
    status = matmul_bias_act::launch_grad<T>(
        dp.at, u.at, w.at, nullptr, du.at, dw.at, dbias.at, mp, first,
        gspace.at, gs.recommended_size, {status.event});
    CHECK(status.status == StatusCode::OK);
    status.event.wait_and_throw();

    const std::vector<double> got_dh = dh.read(), got_dp = dp.read();
    std::vector<double> want_dp(rows * n), want_dbias(n), want_du(rows * width),
        want_dw(width * n), want_dweight(inner);
    for (int b = 0; b < batch; ++b)
      for (int c = 0; c < inner; ++c) {
        double D = 0;
        for (int step = steps - 1; step >= 0; --step) {
          const int r = b * steps + step;
          const double a = sig(got_p[r * n + inner + c]);
          const double prior = step == 0 ? 0 : got_h[(r - 1) * inner + c];
          const double G = got_dh[r * inner + c] + D;
          want_dp[r * n + c] = G * (1 - a);
          want_dp[r * n + inner + c] =
              G * (prior - got_p[r * n + c]) * a * (1 - a);
          D = a * G;
        }
      }
    for (int r = 0; r < rows; ++r) {
      for (int j = 0; j < n; ++j) want_dbias[j] += got_dp[r * n + j];
      for (int k = 0; k < width; ++k)
        for (int j = 0; j < n; ++j) {
          want_du[r * width + k] += got_dp[r * n + j] * w.host[k * n + j];
          want_dw[k * n + j] += got_dp[r * n + j] * u.host[r * width + k];
        }
      double s = 0;
      for (int c = 0; c < inner; ++c)
        s += got_h[r * inner + c] * got_h[r * inner + c];
      for (int c = 0; c < inner; ++c)
        want_dweight[c] += dy.host[r * inner + c] * got_h[r * inner + c] /
                           std::sqrt(s / inner + 1e-6);
    }
    check_all<T>("recurrence's gradient", got_dp, want_dp);
    check_all<T>("bias's gradient", dbias.read(), want_dbias);
    check_all<T>("left gradient", du.read(), want_du);
    check_all<T>("right gradient", dw.read(), want_dw);
    check_all<T>("weight's gradient", dweight.read(), want_dweight);
    // the recurrence's against a difference along a direction, in double
    std::vector<double> ahead = got_p, behind = got_p;
    std::normal_distribution<double> d;
    double along = 0, moved = 0;
    for (size_t i = 0; i < got_p.size(); ++i) {
      const double v = d(gen);
      ahead[i] += 1e-5 * v;
      behind[i] -= 1e-5 * v;
      along += want_dp[i] * v;
    }
    const auto fa = recur(ahead), fb = recur(behind);
    double size = 0;
    for (size_t i = 0; i < fa.size(); ++i) {
      moved += got_dh[i] * (fa[i] - fb[i]) / 2e-5;
      size += std::abs(got_dh[i] * (fa[i] - fb[i]) / 2e-5);
    }
    // (h enters the formula as it was stored)
    CHECK(std::abs(along - moved) <=
          (std::is_same<T, float>::value ? 1e-6 : 0x1p-8) * size);
  }
  (void)hipStreamDestroy(streams[0]);
  (void)hipStreamDestroy(streams[1]);
}

static void refusals() {
  Backend b;
  matmul_bias_act::Params mp{};
  float* none = nullptr;
  auto code = [](const SNNStatus& s) { return s.status; };
  CHECK(code(matmul_bias_act::launch<float>(none, none, none, none, none, none,
                                            mp, b, none, 0)) ==
        StatusCode::InvalidParameter);
  CHECK(code(matmul_bias_act::launch_grad<float>(
            none, none, none, none, none, none, none, mp, b, none, 0)) ==
        StatusCode::InvalidParameter);
  bfloat16* nothing = nullptr;
  linear_recurrence::Params rp{};
  CHECK(code(linear_recurrence::launch<bfloat16>(
            nothing, nothing, nothing, nullptr, nullptr, none, nothing, none, rp,
            b, nothing, 0)) == StatusCode::InvalidParameter);
  residual_norm::Params np{};
  residual_norm::Tensors t{};
  residual_norm::Gradients g{};
  CHECK(code(residual_norm::launch<bfloat16>(t, np, b)) ==
        StatusCode::InvalidParameter);
  CHECK(code(residual_norm::launch_grad<bfloat16>(t, g, np, b, nothing, 0)) ==
        StatusCode::InvalidParameter);
  // elements of the launch's type
  rp.batch = 1;
  rp.steps = 1000;
  rp.channels = 64;
  const size_t half = linear_recurrence::query_workspace_size<bfloat16>(rp)
                          .recommended_size;
  CHECK(half > 0 &&
        linear_recurrence::query_workspace_size<bfloat16>(rp).required_size ==
            0);
}

int main(int argc, char** argv) {
  refusals();
  if (argc < 2 || std::strcmp(argv[1], "--host") != 0) {
    run_block<float>();
    run_block<bfloat16>();
  }
  return report("residual_block");
}
