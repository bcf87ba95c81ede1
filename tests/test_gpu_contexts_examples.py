"""The calls that bitlinear/serve.py's docstring shows, made as they stand there."""
import numpy as np
import pytest
import torch

import bitlinear as bl
import bitlinear.serve as serve
from test_gpu_serve import DEV, dev, rope

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


def test_the_documented_calls():
    n_seqs, n_heads, n_kv_heads, head_dim, n_pages, prompt, max_len = 3, 8, 2, 64, 60, 70, 2049
    rows, pages_each = n_seqs, 33
    rng = np.random.default_rng(51)
    _, _, rope_cos, rope_sin = rope(head_dim, 4000)
    q, k, v = (dev(rng.standard_normal((rows, n * head_dim)).astype(np.float32)) for n in (n_heads, n_kv_heads, n_kv_heads))
    pages = np.full((n_seqs, pages_each), -1, np.int32)
    pages[:, 0] = range(n_seqs)
    names = dict(vars(serve), n_pages=n_pages, n_seqs=n_seqs, n_kv_heads=n_kv_heads, head_dim=head_dim, prompt=prompt,
                 max_len=max_len, max_rows=1, rows=rows, rope_cos=rope_cos, rope_sin=rope_sin, q=q, k=k, v=v,
                 row_start=dev(np.arange(n_seqs + 1, dtype=np.int32)), pos=dev(np.zeros(n_seqs, np.int32)),
                 pages=dev(pages), prompt_pages=dev(np.array([[10, 11]], np.int32)),
                 list_start=dev(np.array([0, rows], np.int32)), prompt_len=dev(np.array([prompt], np.int32)),
                 logits=dev(rng.standard_normal((rows, 100)).astype(np.float32)),
                 u=dev(rng.random(rows).astype(np.float32)))
    lines = [x[4:] for x in serve.__doc__.splitlines() if x.startswith("    ")]
    assert any("paged_attention_account" in x for x in lines)
    for line in lines:
        print(line, flush=True)
        exec(line, names)
    assert names["held"].tolist() == [1] * n_seqs and names["batch"].pos.tolist() == [1] * n_seqs
    assert torch.isfinite(names["o"]).all() and names["ids"].shape == (rows,)
