// The device errors of several translation units as one call reports them.  Plain C++: its test builds it with the
// host compiler.
#pragma once

namespace nnb {

// Word i of `words` holds an error when read(i, where) is not 0; clear(i) resets it.  The first one's status is
// returned, its site in `where`; a reset clears that one alone, and the next call reports the next.
template <class Read, class Clear>
int first_error(int words, bool reset, int* where, Read read, Clear clear) {
  for (int i = 0; i < words; ++i) {
    const int status = read(i, where);
    if (status == 0) continue;
    if (reset) clear(i);
    return status;
  }
  return 0;
}

}  // namespace nnb
