"""Prompts that fill the block table of a rollout engine, on the GPU: they get their token, rows beside them are not disturbed."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHORT = [[1, 2, 3], [400, 5, 77, 9]]


def _engine(kv_dtype, head_dim, max_seq_len=256, **kw):
    from meshy_b200.models.args import ModelArgs
    from meshy_b200.models import build_model
    from meshy_b200.rollout import RolloutEngine

    args = ModelArgs(name="qwen2_5", flavor="lengths_test", dim=512, n_layers=2, n_heads=8, n_kv_heads=2, head_dim=head_dim,
                     ffn_dim=1024, vocab_size=4096, rope_theta=1e6, qkv_bias=True, max_seq_len=2048)
    model = build_model(args, seed=1, device="cuda", dtype=torch.bfloat16)
    return RolloutEngine(args, model=model, device="cuda", max_running=8, max_total_tokens=8192, page_size=64,
                         max_seq_len=max_seq_len, sync_every=4, kv_dtype=kv_dtype, **kw)


@pytest.mark.parametrize("kv_dtype, head_dim, mega", [("auto", 128, "1"), ("auto", 128, "0"), ("auto", 64, "0"), ("int8", 128, "0"),
                                                      ("int8", 64, "0"), ("int4", 128, "0")])
@pytest.mark.parametrize("graphs", [True, False])
def test_full_tables_beside_running_rows(monkeypatch, kv_dtype, head_dim, mega, graphs):
    from meshy_b200.ops._ext import ext

    monkeypatch.setenv("MESHY_MEGA", mega)
    e = _engine(kv_dtype, head_dim, use_cuda_graph=graphs)
    full = [[(11 * i + j) % 4000 + 3 for i in range(n)] for j, n in enumerate((254, 255, 256))]
    before = e.kv.clone() if kv_dtype == "auto" else None
    out = e.generate(full + SHORT, [9, 9, 9, 21, 21], temperature=0.0, ignore_eos=True)
    torch.cuda.synchronize()
    assert int(ext().device_error()) == 0
    assert [len(g.output_ids) for g in out] == [2, 1, 1, 21, 21]
    assert e.blocks.num_free == e.n_pages - 1 and int(e.st["slot"].min()) >= 0 and int(e.st["seq_lens"].max()) <= 256
    # with room behind the prompts (in the same batch, so that every sum has the same order) the tokens are the same
    w = _engine(kv_dtype, head_dim, max_seq_len=1024, use_cuda_graph=graphs)
    want = w.generate(full + SHORT, [2, 1, 1, 21, 21], temperature=0.0, ignore_eos=True)
    for a, b in zip(out, want):
        assert a.output_ids[0] == b.output_ids[0] and len(a.output_ids) == len(b.output_ids)
        assert abs(a.output_logprobs[0] - b.output_logprobs[0]) < 1e-2
    if before is not None:  # pages that no request had are as they were (the last pages of the pool; page 0 is the trash page)
        used = {p for p in range(1, 40)}
        rest = [p for p in range(e.n_pages) if p not in used and p != 0]
        assert rest and torch.equal(e.kv[:, :, rest], before[:, :, rest])
    with pytest.raises(ValueError, match="longer than the 256"):
        e.submit([1] * 257, 3)
