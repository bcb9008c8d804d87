"""How ``prefix_attention`` splits a call, read from its workspace on the CPU: a call that reads prompt and
own keys in one pass needs none, one that stacks all rows against the prompt joins two parts at least."""

from __future__ import annotations

BIG = 1 << 40  # an address nothing dereferences


def _need(fcv, tokens, batch, max_q, prefix, heads=32, kv_heads=8, dim=128, keys=1000, cu=True):
    row = heads * dim
    args = fcv._lib.FcvLmAttention(
        q=BIG, prefix_k=BIG, prefix_v=BIG, k_cache=BIG, v_cache=BIG, cu_q=BIG if cu else None,
        lengths=BIG, out=BIG, q_row=row, q_head=dim, out_row=row, out_head=dim,
        pk_row=kv_heads * dim, pk_head=dim, pv_row=kv_heads * dim, pv_head=dim,
        k_session=keys * kv_heads * dim, k_row=kv_heads * dim, k_head=dim,
        v_session=keys * kv_heads * dim, v_row=kv_heads * dim, v_head=dim, tokens=tokens, batch=batch,
        n_heads=heads, n_kv_heads=kv_heads, head_dim=dim, prefix_len=prefix, sessions=batch,
        capacity=keys, max_q=max_q, max_length=keys, dtype=1, scale=0.1)
    return fcv._lib.load().fcv_lm_prefix_attention_workspace_bytes(args)


def test_a_mixed_batch_reads_a_long_prompt_once(fcv):
    """One text among 63 single tokens: not every sequence reads the prompt in tiles of its own."""
    two_parts = 2 * 575 * 32 * 128 * 4
    assert _need(fcv, 512 + 63, 64, 512, 8192) >= two_parts
    assert _need(fcv, 300 + 7, 8, 300, 2048, 16, 16, 64) > 0
    # nor do single tokens whose bound on the new tokens is loose
    assert _need(fcv, 64, 64, 64, 8192) > 0


def test_texts_take_one_pass(fcv):
    assert _need(fcv, 4 * 512, 4, 512, 4096, cu=False) == 0
    assert _need(fcv, 2700, 4, 1024, 4096) == 0
    assert _need(fcv, 512 + 63, 64, 512, 64) == 0  # a short prompt costs less than the join
    assert _need(fcv, 64 * 512, 64, 512, 0) == 0   # no prompt
