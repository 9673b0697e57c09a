// The rows of a sequence's new tokens, from two neighbouring numbers of the device's offsets: within 0 .. rows whatever those hold.  Both ends are
// bounded before they are subtracted (the difference of any two ints does not fit an int).  Plain C++, for host and device.
#pragma once

namespace eddlhip {

struct SequenceRows {
    int row0, fresh;  // the first row, and how many (none where `end` lies before `begin`)
};
constexpr SequenceRows sequence_rows(int begin, int end, int rows) {
    const int row0 = begin < 0 ? 0 : begin < rows ? begin : rows;
    const int last = end < row0 ? row0 : end < rows ? end : rows;
    return SequenceRows{row0, last - row0};
}

}  // namespace eddlhip
