"""The workspace of packed prompts holds states of sequences that are cut, and
those have more tokens than a segment."""
import pytest


@pytest.mark.parametrize("sequences", [1, 16, 4096, 65536, 1 << 20])
@pytest.mark.parametrize("heads,dim", [((32, 32), 128), ((32, 8), 128), ((12, 12), 64)])
def test_workspace_of_packed_prompts(sequences, heads, dim):
    from catfuse_b200 import _lib
    lib = _lib.load()
    tokens = 1 << 20
    need = lib.cf_decay_attention_workspace(sequences, tokens, *heads, dim, dim, 1)
    state = heads[1] * dim * dim * 4
    # segments have 256 tokens at least; a table entry of 16 bytes each, 4 bytes a sequence
    segments = tokens // 256
    assert 0 <= need <= 2 * segments * state + 16 * (sequences + segments) + 4 * (sequences + 1) + 16
    if sequences >= 65536:  # 16 tokens or fewer each: 137 GB and more if every sequence had a state
        assert need < 1 << 30
