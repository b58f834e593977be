// C++17 face of the 4-bit products (include/infer/linear_hip.hpp): packs, multiplies,
// compares with sums in 64 bits, and throws on what is refused.  With the argument
// "host" only the parts that need no GPU.  Exit status 0 = all passed.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "infer/linear_hip.hpp"

namespace {

int g_failures = 0;

void expect(bool ok, const char* what) {
  if (ok) return;
  ++g_failures;
  std::printf("FAIL %s\n", what);
}

uint16_t to_bf16(float v) {
  uint32_t b;
  std::memcpy(&b, &v, 4);
  b += 0x7FFFu + ((b >> 16) & 1u);
  return static_cast<uint16_t>(b >> 16);
}
float from_bf16(uint16_t w) {
  const uint32_t b = static_cast<uint32_t>(w) << 16;
  float v;
  std::memcpy(&v, &b, 4);
  return v;
}

template <typename F>
bool throws(F f) {
  try {
    f();
  } catch (const infer::Error& e) {
    return std::string(e.what()).find("w4a16") != std::string::npos;
  }
  return false;
}

constexpr int kRows = 37, kCols = 192, kGroup = 64, kTokens = 3;

struct Case {
  std::vector<int8_t> q;
  std::vector<uint16_t> s, x;
  Case() : q(kRows * kCols), s(kRows * (kCols / kGroup)), x(kTokens * kCols) {
    for (size_t i = 0; i < q.size(); ++i) q[i] = static_cast<int8_t>(i * 7 % 16) - 8;
    for (size_t i = 0; i < s.size(); ++i) s[i] = to_bf16((1 + i % 5) / 64.0f);
    for (size_t i = 0; i < x.size(); ++i) x[i] = to_bf16((static_cast<int>(i * 13 % 29) - 14) / 8.0f);
  }
};

void host_parts(const Case& c) {
  const auto w = infer::hip::pack_w4a16(c.q.data(), c.s.data(), kGroup, kRows, kCols);
  expect(w.weight.size() == 48 * 256 / 2 && w.scales.size() == 48 * 3, "sizes of the padded tiles");
  // row 1, columns 8 .. 15 of the second tile: block b = 1, dword 0
  const size_t at = ((0 * 2 + 1) * 4 + 1) * 256 + 1 * 16;
  for (int i = 0; i < 8; ++i) {
    const int nibble = w.weight[at + ((i >> 1) + 4 * (i & 1)) / 2] >> (4 * (((i >> 1) + 4 * (i & 1)) & 1)) & 15;
    expect(nibble == c.q[kCols + 128 + 8 + i] + 8, "a packed value");
  }
  expect(throws([&] { infer::hip::pack_w4a16(c.q.data(), c.s.data(), 48, kRows, kCols); }), "group 48");
  std::vector<int8_t> out_of_range(c.q);
  out_of_range[5] = 8;
  expect(throws([&] { infer::hip::pack_w4a16(out_of_range.data(), c.s.data(), kGroup, kRows, kCols); }),
         "value 8");
  expect(throws([&] {
           infer::hip::gemv_w4a16(nullptr, nullptr, kGroup, nullptr, nullptr, nullptr, 1, kRows, kCols,
                                  nullptr);
         }),
         "null pointers");
}

template <typename T>
T* upload(const std::vector<T>& h) {
  T* p = nullptr;
  infer::hip::check_hip(hipMalloc(reinterpret_cast<void**>(&p), h.size() * sizeof(T)), "hipMalloc");
  infer::hip::check_hip(hipMemcpy(p, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice), "copy");
  return p;
}

void product(const Case& c) {
  const auto w = infer::hip::pack_w4a16(c.q.data(), c.s.data(), kGroup, kRows, kCols);
  infer::hip::Context ctx;
  uint8_t* dw = upload(w.weight);
  uint16_t *ds = upload(w.scales), *dx = upload(c.x), *dy = upload(std::vector<uint16_t>(kTokens * kRows));
  infer::hip::gemv_w4a16(dw, ds, kGroup, nullptr, dx, dy, kTokens, kRows, kCols, ctx.stream());
  ctx.synchronize();
  std::vector<uint16_t> y(kTokens * kRows);
  infer::hip::check_hip(hipMemcpy(y.data(), dy, y.size() * 2, hipMemcpyDeviceToHost), "copy");
  for (int t = 0; t < kTokens; ++t) {
    for (int n = 0; n < kRows; ++n) {
      double exact = 0;
      for (int k = 0; k < kCols; ++k) {
        exact += static_cast<double>(c.q[n * kCols + k]) * from_bf16(c.s[n * 3 + k / kGroup]) *
                 from_bf16(c.x[t * kCols + k]);
      }
      // products and sums of these small dyadic numbers are exact: one rounding to BF16
      expect(std::fabs(from_bf16(y[t * kRows + n]) - exact) <= std::fabs(exact) / 256, "an output");
    }
  }
  for (void* p : {static_cast<void*>(dw), static_cast<void*>(ds), static_cast<void*>(dx), static_cast<void*>(dy)}) {
    (void)hipFree(p);
  }
}

}  // namespace

int main(int argc, char** argv) {
  const Case c;
  host_parts(c);
  if (argc < 2 || std::string(argv[1]) != "host") product(c);
  std::printf(g_failures ? "%d FAILED\n" : "PASSED\n", g_failures);
  return g_failures ? 1 : 0;
}
