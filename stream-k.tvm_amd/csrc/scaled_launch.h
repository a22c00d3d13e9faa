// Between the C ABI and the units that hold the int8 kernels with scales.  Ids are those of the int8 kernels (kernel_table.h).
#pragma once
#include "launch.h"
#include "tile_scaled_i8.h"

namespace sk {

bool has_scaled_i8(int id);
// hipError_t as int (hipErrorInvalidValue: an id without an instance); co-resident CTAs per CU, 0 without an instance
int launch_scaled_i8(int id, const GemmArgs &a, const Scales &sc, const DevPlan &p, const Workspace &ws, hipStream_t s, const void *bias);
int occupancy_scaled_i8(int id);
bool has_scaled_i8_asm(int id);
int launch_scaled_i8_asm(int id, const GemmArgs &a, const Scales &sc, const DevPlan &p, const Workspace &ws, hipStream_t s, const void *bias);
int occupancy_scaled_i8_asm(int id);

}  // namespace sk
