// The few-row mixture's products on bf16 coefficients.
#include "ckan_few.hpp"

namespace ckan {

void launch_few_bf16(const FewArgs& a, hipStream_t st) {
  a.x_bf16 ? launch_degree<__bf16, __bf16>(a, st) : launch_degree<float, __bf16>(a, st);
}

}  // namespace ckan
