// Words of host memory that kernels write to whose bounded wait ran out: one for each operator that has such waits, and device.
#pragma once

namespace b200ccl::kernels {

enum class WaitsOf : int { WeightGrad = 0, VocabularyLoss = 1 };
constexpr int kWaitsOf = 2;

unsigned* wait_status_word(WaitsOf what, int device);
// Whether a wait ran out on `device` since this was last asked.
bool waits_failed(WaitsOf what, int device);

}  // namespace b200ccl::kernels
