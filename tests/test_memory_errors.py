"""The memory-over-ticks operators' errors on the host. Without a GPU."""
import pytest

from flyguy_b200 import memory, native


def test_a_refused_size_is_refused_in_the_same_words_again():
    """A workspace's size is kept from call to call; a refusal's words are the refusal's each time, also after a call that went
    well."""
    good, bad = (1, 8, 2, 2, 64, 64, 0), (1, 8, 2, 2, 300, 64, 0)
    for _ in range(3):
        with pytest.raises(native.FlyguyError, match="dim and value_dim must be 1 to 256"):
            memory._room(memory._decay_room(bad, False, False), None)
        assert native.lib().fg_decay_work(memory._DECAY.pack(*(0,) * 38, *good, 1.0, 0, 0), 0) == 0
        assert native.lib().fg_mem_last_error() == b""
