"""CPU checks of the gated scan's C entry."""


def test_more_sequences_than_tokens_need_a_status_word():
    """Without one every sequence is active and needs a token; with one the sequence count is a capacity."""
    from flashrwkv2_b200 import _lib

    lib = _lib.load()
    assert lib.frwkv_sm100_gated_scan(16, 16, 0, 16, 16, 64, 16, 64, 0, 16, 5, 4, 64, 0, 0, 0, 0, 0) != 0
    assert "at least 5 token" in _lib.last_error()
