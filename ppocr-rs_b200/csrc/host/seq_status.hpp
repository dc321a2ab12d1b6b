// The words of page-locked host memory that the sequence operators' kernels
// report in.
#pragma once

namespace ppocr {

// Takes what a word holds and leaves 0, in one step: a report that a kernel on
// another stream writes meanwhile is either taken or still there.
inline int take_status(int* word) { return __atomic_exchange_n(word, 0, __ATOMIC_SEQ_CST); }

}  // namespace ppocr
