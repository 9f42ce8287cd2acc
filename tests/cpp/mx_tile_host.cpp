// Host check of where the tiles of 4-bit rows read (vectoraccelerate_amd/csrc/va_mx_tile.hpp): every lane of every stage's load, at rows and
// pitches of all kinds, either fails the descriptor's range check, which compares the lane's own offset, or reads inside the rows; and
// what is multiplied is what belongs there.
#include <cstdio>
#include <vector>

#include "../../vectoraccelerate_amd/csrc/va_mx_tile.hpp"

using namespace va;

static long failures = 0, loads = 0;

// one load of `width` bytes at lane offset `off`: whether it is made; it must stay in `records`
static bool made(uint32_t off, uint32_t width, uint32_t records, const char* what, uint32_t groups, uint32_t rows, uint32_t pitch, uint32_t stage) {
    ++loads;
    if (off >= records) return false;
    if (off + width > records && ++failures <= 20)
        std::printf("FAIL %s: groups %u, rows %u, pitch %u, stage %u: offset %u of %u\n", what, groups, rows, pitch, stage, off, records);
    return true;
}

template <int GS>
static void check(uint32_t tile, bool items, uint32_t groups, uint32_t rows, uint32_t pad) {
    const uint32_t pitch = rows == 1 ? 0 : groups * kMxCodes + 16 * pad, scale_pitch = rows == 1 ? 0 : groups * kMxScales + 4 * pad, stages = (groups + GS - 1) / GS;
    for (uint32_t s = 0; s < stages; ++s)
        for (uint32_t row = 0; row < tile; ++row) {
            const uint32_t source = items ? mx_item_of(row) : row;
            for (uint32_t c = 0; c < 4 * GS; ++c) {
                const uint32_t off = mx_stage_offset(mx_code_offset<GS>(row, c, source, pitch), s, GS * kMxCodes);
                const bool there = made(off, 16, mx_records(rows, pitch, groups, kMxCodes), "codes", groups, rows, pitch, s);
                const uint32_t chunk = c ^ mx_swizzle<GS>(row);  // of the stage
                if (source < rows && s * GS + chunk / 4 < groups && (!there || off != source * pitch + s * GS * kMxCodes + 16 * chunk) && ++failures <= 20)
                    std::printf("FAIL codes: groups %u, rows %u: row %u, chunk %u, stage %u is read from %u\n", groups, rows, source, chunk, s, off);
            }
            for (uint32_t g = 0; g < GS; ++g) {
                const uint32_t off = mx_stage_offset(mx_scale_offset(g, source, scale_pitch), s, GS * kMxScales);
                const bool there = made(off, 4, mx_records(rows, scale_pitch, groups, kMxScales), "scales", groups, rows, scale_pitch, s);
                if (source < rows && s * GS + g < groups && (!there || off != source * scale_pitch + 4 * (s * GS + g)) && ++failures <= 20)
                    std::printf("FAIL scales: groups %u, rows %u: row %u, group %u is read from %u\n", groups, rows, source, s * GS + g, off);
            }
        }
}

int main() {
    for (uint32_t groups : {1u, 2u, 3u, 4u, 5u, 6u, 7u, 11u, 12u, 13u, 511u, 512u})
        for (uint32_t pad : {0u, 1u, 5u}) {
            if (groups * kMxCodes + 16 * pad > 65536) continue;
            for (uint32_t rows : {1u, 2u, 63u, 64u, 65u, 127u, 128u, 200u, 255u, 256u}) {
                check<2>(256, true, groups, rows, pad);
                check<1>(256, true, groups, rows, pad);
                if (rows <= 128) check<2>(128, false, groups, rows, pad);
                if (rows <= 64) check<1>(64, false, groups, rows, pad);
            }
        }
    std::printf("mx_tile_host: %ld loads, %ld failures%s\n", loads, failures, failures ? "" : ", ok");
    return failures != 0;
}
