"""CPU tests of the sizes at which the batched serving ops are refused before any device work."""
import bitlinear as bl
from test_serve_host import attention, batch, cache


def test_attention_over_one_grid_of_threads():
    """2^32 threads and more are refused as a shape: 2^23 workgroups of 512 (sequences of up to 512
    tokens), 2^24 of 256."""
    most = dict(n_seqs=1 << 20, rows=1 << 20, max_rows=1, max_pages=64)
    assert attention(c=cache(n_kv_heads=8), b=batch(max_len=512, **most), nh=8) == bl.BTL_ERR_SHAPE
    assert b"too large for one launch" in bl.lib.btl_last_error()
    assert attention(c=cache(n_kv_heads=16), b=batch(max_len=600, **most), nh=16) == bl.BTL_ERR_SHAPE
    # one head less: past the check, up to the buffers that are not there
    for nkv, length in ((7, 512), (5, 600)):
        assert attention(c=cache(n_kv_heads=nkv, k=None), b=batch(max_len=length, **most), nh=nkv) == bl.BTL_ERR_LAYOUT
