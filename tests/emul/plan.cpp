// The fused linear layer's choice of kernels (tempo_amd/csrc/linear_plan.h), CPU only.
#include "../../tempo_amd/csrc/linear_plan.h"

extern "C" {

// kernel, xi, xj, ti, tj, split into out[6]; 0 where the product is refused
int emul_plan_product(long long I, long long J, long long K, int al, int bl, int dtype, int direct,
                      long long* out) {
  Product p = {};
  if (!plan_product(I, J, K, al, bl, dtype, direct != 0, &p)) return 0;
  const bool tiled = p.kernel != FEW && p.kernel != THIN;
  const long long r[6] = {p.kernel, p.xi, p.xj, tiled ? p.ti : 0, tiled ? p.tj : 0, p.split};
  for (int n = 0; n < 6; ++n) out[n] = r[n];
  return 1;
}

int emul_streamable(long long address, long long ld, int layout, long long rows, long long K,
                    int size) {
  return streamable((const void*)(uintptr_t)address, ld, layout, rows, K, size);
}

long long emul_product_bytes(long long I, long long J, long long K, int al, int bl, int dtype) {
  long long bytes;
  return product_bytes(I, J, K, al, bl, dtype, &bytes) ? bytes : -1;
}

}  // extern "C"
