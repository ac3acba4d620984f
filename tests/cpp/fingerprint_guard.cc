// argv[1]: a call of mirage::search on a graph with an operator that has no fingerprint ("plain": on one without).
#include "mirage/kernel/graph.h"
#include "mirage/search/checkpoint.h"
#include "mirage/search/verify.h"

#include <cstdio>
#include <cstring>

using namespace mirage;

int main(int argc, char **argv) {
  char const *what = argc > 1 ? argv[1] : "";
  kernel::Graph plain, with;
  plain.exp(plain.new_input({4, 64}, type::DT_FLOAT16, layout::DmemRowMajor));
  auto x = with.new_input({4, 2, 64}, type::DT_FLOAT16, layout::DmemRowMajor);
  auto positions = with.new_input({4}, type::DT_INT32, layout::DmemRowMajor);
  auto angles = with.new_input({2, 32}, type::DT_DOUBLE, layout::DmemRowMajor);
  with.exp(with.rotary(x, positions, angles));
  std::vector<uint8_t> equal;
  if (std::strcmp(what, "graph") == 0) {
    search::fingerprint_graph(with, 1);
  } else if (std::strcmp(what, "candidate") == 0) {
    search::verify_batch({&plain, &with}, search::graph_outputs(plain), 1, equal);
  } else if (std::strcmp(what, "reference") == 0) {
    search::verify_batch_begin({&plain}, search::graph_outputs(with), 1, &with);
  } else if (std::strcmp(what, "outputs") == 0) {
    search::verify_batch({&plain}, {with.operators[3]->output_tensors[0]}, 1, equal);
  } else if (std::strcmp(what, "ask") == 0) {
    std::printf("%d %d\n", search::has_fingerprints(plain) ? 1 : 0, search::has_fingerprints(with) ? 1 : 0);
  } else if (std::strcmp(what, "plain") == 0) {
    search::fingerprint_graph(plain, 1);
  }
  return 0;
}
