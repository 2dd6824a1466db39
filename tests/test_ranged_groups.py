"""The plan of calls over shared prefixes, as the sizes of their workspaces show it (without a GPU: of 256 CUs)."""
from __future__ import annotations

import torch

from flour_amd import ops


def pieces(num_seqs, num_groups, max_rows, rows, heads, kv_heads, dim, max_kv, max_shared, dtype):
    """Pieces of a (row, head) that a call has room for: a maximum, a sum and dim accumulators each."""
    return ops.shared_workspace_bytes(num_seqs, num_groups, max_rows, rows, heads, kv_heads, dim, max_kv,
                                      max_shared, dtype) // (rows * heads * (dim + 2) * 4)


def test_sequences_without_a_prefix_have_pieces_like_the_prefixes():
    """64 chats, prefixes of up to 16,384 positions: one of them can have all its 16,640 to itself, 260 tiles of
    64, where a prefix is cut into 16 pieces."""
    assert pieces(64, 1, 1, 64, 32, 8, 128, 16640, 16384, torch.bfloat16) >= 2 * 15
    assert pieces(32, 1, 8, 170, 32, 8, 128, 5120, 4096, torch.bfloat16) >= 2 * 4  # drafted rows
    assert pieces(16, 1, 1, 16, 8, 8, 64, 2304, 2048, torch.float32) >= 2 * 7


def test_packed_calls_of_one_row_a_sequence_are_not_judged_as_steps():
    """Their other way is row tiles, not the decode stream: 64 fp32 chats over 1,024 + 256 positions take 107 us
    on those and 40 with their prefix for all."""
    assert pieces(64, 1, 1, 65, 8, 8, 64, 1280, 1024, torch.float32) >= 2  # (a row of padding: no step)
    assert pieces(64, 1, 1, 64, 8, 8, 64, 1280, 1024, torch.float32) >= 2  # (either)
    assert pieces(5000, 10, 1, 5000, 8, 8, 64, 1280, 1024, torch.float32) >= 2  # (more than the stream takes)
