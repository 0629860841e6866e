// Calls of the training operators that are refused before any CUDA call, on
// engine and buffer objects made here: buffers on another GPU than the engine,
// which needs no second GPU that way (tests/test_training_ops_other_gpu.py).
#include <cstdio>
#include <cstring>

#include "engine.h"

namespace {

int failures = 0;

void want(const char* what, int rc) {
  const bool ok = rc == EB_INVALID_ARGUMENT && std::strstr(eb_last_error(), "on another GPU");
  if (!ok) std::printf("%s: status %d, \"%s\"\n", what, rc, eb_last_error());
  failures += !ok;
}

// A buffer object over no memory: its address is only compared.
eb_buf buffer(size_t at, size_t len, int dtype = EB_F32, int device = 1) {
  eb_buf b;
  b.ptr = reinterpret_cast<void*>(4096 + at);
  b.len = len;
  b.dtype = dtype;
  b.device = device;
  return b;
}

}  // namespace

int main() {
  eb_engine e;
  e.device = 1;
  eb_buf b[8];
  auto fresh = [&](int i) {  // all on GPU 1 but number i
    for (int j = 0; j < 8; j++) b[j] = buffer(4096 * j, 64, EB_F32, j == i ? 0 : 1);
  };
  for (int i = 0; i < 6; i++) {
    fresh(i);
    want("layer norm", eb_layer_norm(&e, b + 0, 8, 8, 0, b + 1, b + 2, 1e-5f, b + 3, 0, b + 4, b + 5));
  }
  for (int i = 0; i < 8; i++) {
    fresh(i);
    want("layer norm backward", eb_layer_norm_backward(&e, b + 0, 0, b + 1, 0, 8, 8, b + 2, b + 3,
                                                       b + 4, b + 5, 0, b + 6, b + 7));
  }
  for (int i = 0; i < 5; i++) {
    fresh(i);
    b[2].dtype = EB_U32;
    want("cross entropy", eb_linear_ce(&e, b + 0, 8, 8, 0, b + 1, 8, 0, b + 2, 1.0f, b + 3, b + 4));
  }
  for (int i = 0; i < 7; i++) {
    fresh(i);
    b[2].dtype = EB_U32;
    want("cross entropy backward", eb_linear_ce_backward(&e, b + 0, 8, 8, 0, b + 1, 8, 0, b + 2,
                                                         1.0f, b + 3, b + 4, b + 5, 0, b + 6, 0));
  }
  for (int i = 0; i < 7; i++) {
    fresh(i);
    b[2].dtype = b[3].dtype = EB_F8;
    b[6].dtype = EB_BF16;
    const eb_adamw_tensor t{b + 0, b + 1, b + 2, b + 3, b + 4, b + 5, b + 6, 0.0};
    eb_adamw* plan = nullptr;
    want("adamw", eb_adamw_create(&e, &t, 1, &plan));
  }
  std::printf("%d failures\n", failures);
  return failures != 0;
}
