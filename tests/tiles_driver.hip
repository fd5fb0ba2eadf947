// tiles_driver.hip — which tiles and splits the products of a call take, by the rules that the calls themselves use.  Host code
// only: it is compiled without a device pass and launches nothing.
//
// A line "ff T n width inner grad" is answered by those of the projections, and with grad of dx and dW, and
// whether the two share a launch; "ortho K batch rows cols" (K: fast or exact) by those of A, B and X.  Each is shape/splits.
#include "ec_ff.hip"
#include "ec_ortho.hip"

#include <iostream>
#include <string>

namespace {

std::string text(const ec::Choice& c) {
  static const char* names[] = {"large", "middle", "least"};
  return std::string(names[c.shape]) + "/" + std::to_string(c.splits.n);
}

template <typename T>
void ff(uint64_t n, uint64_t width, uint64_t inner, bool grad) {
  std::cout << text(ec::choose_ff<T>(n, width, inner));
  if (grad) {
    const uint64_t low = sizeof(T) < 4 && n <= ec::kFewRows ? 2 : 1;
    const ec::Choice dx = ec::choose_sum<T>(n, width, inner, 2 * low, 1), dw = ec::choose_sum<T>(inner, width, n, low, 2);
    std::cout << ' ' << text(dx) << ' ' << text(dw);
  }
  std::cout << '\n';
}

template <typename In>
void ortho(uint32_t batch, uint32_t rows, uint32_t cols) {
  const uint32_t side = std::min(rows, cols), other = std::max(rows, cols);
  std::cout << text(ec::choose_ns<In>(side, side, other, batch, ec::kGram)) << ' '
            << text(ec::choose_ns<In>(side, side, side, batch, ec::kPoly)) << ' '
            << text(ec::choose_ns<In>(rows, cols, side, batch, ec::kNext)) << '\n';
}

}  // namespace

int main() {
  std::string op, type;
  while (std::cin >> op >> type) {
    if (op == "ff") {
      uint64_t n, width, inner;
      int grad;
      std::cin >> n >> width >> inner >> grad;
      if (type == "fp32")
        ff<float>(n, width, inner, grad);
      else if (type == "bf16")
        ff<ec::bf16_t>(n, width, inner, grad);
      else
        ff<ec::fp16_t>(n, width, inner, grad);
    } else {
      uint32_t batch, rows, cols;
      std::cin >> batch >> rows >> cols;
      if (type == "fast")
        ortho<ec::fp16_t>(batch, rows, cols);
      else
        ortho<ec::pair_t>(batch, rows, cols);
    }
  }
}
