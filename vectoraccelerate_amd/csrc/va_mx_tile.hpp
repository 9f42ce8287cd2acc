// va_mx_tile.hpp — where the tiles' direct loads of coded rows read (va_mx.hip).  No HIP dependency: a host program checks that no lane
// reads past the rows that it is given.
//
// A descriptor covers a tile's rows up to the end of the last one.  Lanes of rows that are not there, and of a group that the last row does
// not have, must fail its range check, and the check may leave a load's scalar offset out; so a stage's place in the row is part of
// the lane's own offset.
#pragma once

#include <cstdint>

namespace va {

constexpr uint32_t kMxCodes = 64, kMxScales = 4;  // bytes of a group of 128 values

// The item of a wave's 64 that lies in LDS row r of them: two neighbours go to one lane.
constexpr uint32_t mx_item_of(uint32_t r) { return r / 64u * 64u + r % 32u * 2u + r % 64u / 32u; }
// What the 16-byte chunks of an LDS row of GS groups are turned by.
template <int GS>
constexpr uint32_t mx_swizzle(uint32_t row) {
    return (GS == 1 ? row >> 2 : row >> 1) & uint32_t(4 * GS - 1);
}
// Bytes from the tile's first row to what physical chunk c of LDS row `row` takes of the first stage: from row `source`.
template <int GS>
constexpr uint32_t mx_code_offset(uint32_t row, uint32_t c, uint32_t source, uint32_t pitch) {
    return source * pitch + 16u * (c ^ mx_swizzle<GS>(row));
}
// The same for the four scale bytes of a stage's group g.
constexpr uint32_t mx_scale_offset(uint32_t g, uint32_t source, uint32_t pitch) { return source * pitch + kMxScales * g; }
// A lane's offset in stage `stage`, of `bytes` a row.
constexpr uint32_t mx_stage_offset(uint32_t first, uint32_t stage, uint32_t bytes) { return first + stage * bytes; }
// What the descriptor of `rows` rows covers, each of `groups` groups of `bytes`.
constexpr uint32_t mx_records(uint32_t rows, uint32_t pitch, uint32_t groups, uint32_t bytes) { return (rows - 1) * pitch + groups * bytes; }

}  // namespace va
