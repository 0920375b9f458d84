#pragma once
// Where a lane's chunk of a k-step lies in its operand's row, for the input-gradient GEMMs: c = the chunk's first element within the step, k0 =
// the step's first element, K = the row's length (a multiple of 8, so a chunk of 4 or 8 elements is all inside or all outside).  A
// chunk outside reads elements of the row that are there; what it read is masked on its way to LDS.  Plain C++, so that the host can check
// every lane: row + chunk must end inside the operand, also for rows shorter than a step (K = 8, 16, 24) and steps past the row's end.

// the row's part of a lane's pointer: the row itself, or the last one
constexpr int qbs_row(int first, int row, int rows) { return first + row < rows ? first + row : rows - 1; }
// wide kernel: the pointer holds the chunk's place in the first step, or 0 where the row is shorter than that ...
constexpr int qbs_chunk0(int c, int K) { return c < K ? c : 0; }
// ... and a load adds the step's place
constexpr int qbs_step(int c, int k0, int K) { return k0 + c < K ? k0 : 0; }
// narrow kernel: from the row's first element (its pointers hold c, hence the - c)
constexpr int qbs_chunk(int c, int k0, int K) { return k0 + c < K ? k0 + c : 0; }
constexpr int qbs_chunk_from_c(int c, int k0, int K) { return k0 + c < K ? k0 : -c; }
