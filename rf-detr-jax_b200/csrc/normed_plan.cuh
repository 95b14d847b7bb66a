// How the lanes of a warp share a row of the normed rotary positions: host arithmetic alone, no device code.
#pragma once

namespace rfdetr {

// How a lane finds the partners of its channels: it holds both, from two pieces half apart (kPaired) or from one
// (kInterleaved), or they meet through shared memory (kExchange).
enum NormMode { kPaired, kInterleaved, kExchange };

struct NormPlan {
    NormMode mode;
    int vec;     // values to a piece
    int pieces;  // of a row
    int each;    // to a lane at most
    int lanes;   // that hold a row
};

// Rows of D channels (256 at most), of which 2 half turn; whole: all are read in pieces of 16 bytes.  Sixteen bf16
// values (eight float32) to a lane, so that what a row costs besides them is shared; a paired piece is two vectors
// where it turns and one where it does not, so that float32 rows that turn in a small part have up to 48 pieces: where
// they pass a warp's 32 lanes a lane has two.  Read value by value, eight to a lane.
inline NormPlan plan_normed(int value_bytes, int D, int half, bool interleaved, bool whole) {
    NormPlan p{};
    p.vec = whole ? 16 / value_bytes : 1;
    p.mode = !whole ? kExchange : interleaved ? kInterleaved : half % p.vec == 0 ? kPaired : kExchange;
    p.pieces = p.mode == kPaired ? half / p.vec + (D - 2 * half) / p.vec : D / p.vec;
    p.each = !whole ? 8 : p.mode == kPaired && p.pieces <= 32 ? 1 : 2;
    p.lanes = (p.pieces + p.each - 1) / p.each;
    return p;
}

}  // namespace rfdetr
