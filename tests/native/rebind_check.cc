// Host-only: which tensors the orthogonalised updates are asked to move after a parameter was bound to its caller's own.  The device is device_standin.cc.
#include <cstdio>
#include <vector>

#include "engine.h"

static std::vector<cavs_ortho_desc> asked;
extern "C" int cavs_ortho_update_in_out(int, int count, const cavs_ortho_desc *d, const cavs_ortho_options *, void *, size_t, void *) {
  asked.assign(d, d + count);
  return 0;
}

int main() {
  cavs_session_config cfg{};
  cfg.model = CAVS_MODEL_TREELSTM, cfg.opt = CAVS_OPT_BATCHING, cfg.V = 10, cfg.E = 8, cfg.H = 32, cfg.C = 5, cfg.optimizer = CAVS_OPTIMIZER_ORTHO;
  cavs::Engine e(cfg);
  const size_t nw = 8 * 4 * 32, nu = 4 * 32 * 32;
  std::vector<float> w(nw), gw(nw), u(nu), gu(nu), x(3), labels(3);
  const int graph[] = {2, 2, -1};
  int wrong = 0;
  auto owns = [](const std::vector<float> &v, const void *p) { return p >= v.data() && p < v.data() + v.size(); };
  auto step = [&](bool w_bound, bool u_bound) {
    asked.clear();
    e.step(graph, 1, 3, x.data(), labels.data(), false, true, 0.1f);
    if (asked.size() != 8) wrong++;
    for (size_t i = 0; i < asked.size(); i++) {  // four blocks of W, four of U
      const bool in_w = i < 4;
      if (owns(in_w ? w : u, asked[i].W) != (in_w ? w_bound : u_bound) || owns(in_w ? gw : gu, asked[i].G) != (in_w ? w_bound : u_bound)) {
        std::printf("block %zu: W %p G %p\n", i, (void *)asked[i].W, asked[i].G);
        wrong++;
      }
    }
  };
  step(false, false);
  e.bind_param("W", w.data(), gw.data());
  step(true, false);
  e.bind_param("U", u.data(), gu.data());
  step(true, true);
  std::printf("%d wrong\n", wrong);
  return wrong != 0;
}
