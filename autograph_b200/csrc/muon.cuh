// What the model layer takes of the Newton-Schulz steps beside the C entries.
#pragma once

#include <vector>

#include "common.cuh"

namespace ag {

// The sizes that ag_muon_update checks, and its workspace, ahead of the first update: after this an update of matrices of these
// sizes is not refused and asks for no memory.  The matrices' pointers are not looked at.
int muon_prepare(ag_device *dev, ag_dtype dtype, const std::vector<ag_muon_matrix> &matrices, int steps);

}  // namespace ag
