"""CPU tests of the largest calls that the 8-bit operators take."""
import pytest

from moba_hip.ops import _lib
from moba_hip.quantized import _attention_work

MILLION = 2 ** 20
# the largest number of rows of 2 kv heads: 512 threads join each row and kv head, and 95
# times `group` workgroups wait for entries of many parts
LAST = {1: (2 ** 23 - 96) // 2, 2: (2 ** 23 - 191) // 2, 16: (2 ** 23 - 1521) // 2}


@pytest.mark.parametrize("group", LAST)
def test_the_threads_of_a_launch_bound_an_attention(group):
    """2^32 threads are more than a launch holds."""
    work = _lib.load().moba_hip_quantized_attention_work
    rows = LAST[group]
    assert work(rows, 2 * group, 2, 64, 0, 0, 32) > 0
    assert work(rows + 1, 2 * group, 2, 64, 0, 0, 32) == -1
    assert _attention_work(rows, 2 * group, 2, 64, 0, 0, 32) == work(rows, 2 * group, 2, 64, 0, 0, 32)
    with pytest.raises(ValueError, match="blocks of 16 heads"):
        _attention_work(rows + 1, 2 * group, 2, 64, 0, 0, 32)


@pytest.mark.parametrize("args", [
    (MILLION, 8, 8, 64, 0, 0, 32), (MILLION, 8, 8, 64, 4, 16, 32),     # 2^23 entries
    (2 ** 16, 2 ** 15, 1, 64, 0, 0, 32),                               # 2^31 heads
    (2 ** 13, 8, 8, 64, 0, 0, 2 ** 22),                                # 2^31 units and two an entry
    (1, 8, 8, 64, 0, 0, 0x7fff0001), (2 ** 33, 8, 8, 64, 0, 0, 32)])
def test_attentions_that_pass_a_counter(args):
    with pytest.raises(ValueError, match="2\\^31"):
        _attention_work(*args)


def test_the_entry_refuses_what_the_workspace_refuses():
    """Before anything is launched."""
    lib = _lib.load()
    for rows, hq in ((LAST[2] + 1, 4), (2 ** 29, 4), (2 ** 30, 4)):
        rc = lib.moba_hip_quantized_attention(64, 0, rows, hq, 2, 64, 1.0, 0, 64, 64, 64, 64, 4, 16, 64, 2, 2, 64, 64,
                                              0, 32, None, 0, 0, 64, 64, 64, None)
        assert rc == _lib.MOBA_ERR_ARG and "threads of a launch" in lib.moba_hip_last_error().decode()


@pytest.mark.parametrize("hkv,d", [(2 ** 23, 64), (2 ** 21, 256)])
def test_an_item_of_the_means_that_no_launch_holds(hkv, d):
    """64 threads for 8 dims of a kv head: 2^26 of these are 2^32."""
    lib = _lib.load()
    rc = lib.moba_hip_quantized_means(0, 64, 64, 1, 16, hkv, d, 64, 2, 1, 64, 64, 1, 0, 8, 0, 64, 2, None)
    assert rc == _lib.MOBA_ERR_ARG and "quantized_means" in lib.moba_hip_last_error().decode()


def test_the_ends_of_scale():
    """The entry takes both ends: what it refuses here is the length."""
    lib = _lib.load()
    for scale, word in ((2.0 ** -126, "max_length"), (1e30, "max_length"), (1e30 * (1 - 2.0 ** -50), "max_length"),
                        (2.0 ** -127, "scale"), (1.1e30, "scale"), (float("inf"), "scale")):
        rc = lib.moba_hip_quantized_attention(64, 0, 1, 4, 2, 64, scale, 0, 64, 64, 64, 64, 4, 16, 64, 2, 2, 64, 64,
                                              0, 0, None, 0, 0, 64, 64, 64, None)
        assert rc == _lib.MOBA_ERR_ARG and f"{word} must be" in lib.moba_hip_last_error().decode()


def test_selected_chunks_have_one_block_of_heads_an_entry():
    """However long the table: a workspace for chunks that each head selects is made for what
    they hold, and two blocks of heads would have twice the partials."""
    work = _lib.load().moba_hip_quantized_attention_work
    assert work(64, 32, 1, 128, 4, 64, 131072) == work(64, 32, 1, 128, 4, 64, 8192)
    assert work(64, 32, 1, 128, 0, 0, 131072) > 1.9 * work(64, 32, 1, 128, 0, 0, 8192)
