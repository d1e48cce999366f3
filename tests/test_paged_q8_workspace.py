"""The workspace of many rows over 8-bit pages: a copy of the keys in fp16, of
one sequence or of as many as 2 GiB hold, beside the partial results of a few
ranges of the keys (CPU)."""
import pytest

from npu_comp_b200 import _lib

GIB2 = 1 << 31


def one(ctx, KV, hd):
    """Bytes of one sequence's copy: K and V, two scales for 16 keys, ids and length."""
    keys = (ctx + 127) // 128 * 128
    return keys * KV * hd * 4 + keys // 16 * KV * 8 + keys // 128 * 4 + 4


def parts(total, H, hd, ranges=4):  # (128 at most: where the rows fill few of the SMs)
    return ranges * total * H * (hd * 4 + 8)


@pytest.mark.parametrize("batch,total,ctx,H,KV,hd,ranges", [
    (64, 6400, 131072, 32, 8, 128, 4), (16, 4000, 131072, 32, 8, 128, 4), (4096, 100000, 32768, 8, 8, 128, 4),
    (65535, 65535, 1 << 20, 1, 1, 16, 128), (300, 9000, 8192, 32, 32, 64, 4),
])
def test_many_sequences(libnpub_path, batch, total, ctx, H, KV, hd, ranges):
    query = _lib.load().npub_attention_paged_q8_workspace
    for max_new in (0, min(total, 1 << 20)):
        n = query(batch, total, max_new, ctx, H, KV, hd)
        assert one(ctx, KV, hd) <= n <= max(GIB2, one(ctx, KV, hd)) + parts(total, H, hd, ranges) + 1024


def test_small_calls_hold_all_their_sequences(libnpub_path):
    query = _lib.load().npub_attention_paged_q8_workspace
    n = query(16, 4000, 500, 8192, 32, 8, 128)
    assert 16 * one(8192, 8, 128) <= n <= 16 * one(8192, 8, 128) + parts(4000, 32, 128) + 1024
    # one sequence is held whatever its length
    assert query(1, 4000, 4000, 1 << 21, 32, 8, 128) >= one(1 << 21, 8, 128) > GIB2
