"""The drafted step's arguments are checked before a device sees them: what a kernel reads or writes for each row, node
or sequence has to be there."""
import pytest
import torch

from ferrisinfer_amd import DTYPE_BF16, FerrisError, kernel


def context():
    """A context without a device: what reaches the library is refused there as InvalidConfig."""
    ctx = object.__new__(kernel.Context)
    ctx.lib, ctx.handle = kernel.load(), None
    return ctx


def i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def f(*shape):
    return torch.zeros(shape)


def q(*shape):
    return torch.zeros(shape, dtype=torch.int64)


# an entry's arguments in order, for two sequences of six rows in all
CALLS = {
    "tree_plan": dict(parents=i(6), cu_seqlens=i(3), context_lens=i(2), max_query_len=4, mask_out=q(6, 1), positions_out=i(6)),
    "attn_tree_paged": dict(q=f(6, 4, 32), k_cache=f(4, 2, 16, 32), v_cache=f(4, 2, 16, 32), kv_dtype=DTYPE_BF16, block_tables=i(2, 4),
                            cu_seqlens=i(3), context_lens=i(2), tree_mask=q(6, 1), max_query_len=4, max_context_len=64, num_kv_heads=2,
                            block_size=16, num_blocks=4, scale=0.2, out=f(6, 4, 32)),
    "verify_drafts": dict(logits=f(6, 50), tokens=i(6), parents=i(6), cu_seqlens=i(3), max_query_len=4, temperature=f(2), accept_u=f(6),
                          pick_u=f(2), draft_probs=f(6, 50), distinct=False, tokens_out=i(2, 4), path_out=i(2, 3), count_out=i(2),
                          prob_out=f(2)),
    "kv_keep_path": dict(k_caches=[f(4, 2, 16, 32)], v_caches=[f(4, 2, 16, 32)], kv_dtype=DTYPE_BF16, block_tables=i(2, 4), cu_seqlens=i(3),
                         context_lens=i(2), path=i(2, 3), num_blocks=4, block_size=16, num_kv_heads=2, head_dim=32),
}
REFUSED = [
    ("tree_plan", dict(positions_out=i(5)), "InvalidShape"),
    ("tree_plan", dict(mask_out=q(5, 1)), "InvalidShape"),
    ("tree_plan", dict(mask_out=i(6, 1)), "InvalidType"),
    ("tree_plan", dict(mask_out=q(1, 6).T), "InvalidConfig"),  # (one word a row: contiguous)
    ("tree_plan", dict(mask_out=q(2, 6).T), "InvalidLayout"),
    ("tree_plan", dict(cu_seqlens=i(2)), "InvalidShape"),
    ("tree_plan", dict(parents=q(6)), "InvalidType"),
    ("tree_plan", dict(context_lens=i(4)[::2]), "InvalidLayout"),
    ("attn_tree_paged", dict(out=f(5, 4, 32)), "InvalidShape"),
    ("attn_tree_paged", dict(out=f(6, 4, 64)), "InvalidShape"),
    ("attn_tree_paged", dict(out=f(6, 4, 32).half()), "InvalidType"),
    ("attn_tree_paged", dict(q=f(4, 6, 32).transpose(0, 1)), "InvalidLayout"),
    ("attn_tree_paged", dict(tree_mask=q(5, 1)), "InvalidShape"),
    ("attn_tree_paged", dict(block_tables=i(1, 4)), "InvalidShape"),
    ("attn_tree_paged", dict(block_tables=i(4, 2).T), "InvalidLayout"),
    ("attn_tree_paged", dict(cu_seqlens=q(3)), "InvalidType"),
    ("verify_drafts", dict(logits=f(50, 6).T), "InvalidLayout"),
    ("verify_drafts", dict(logits=f(6, 50).double()), "InvalidType"),
    ("verify_drafts", dict(draft_probs=f(6, 49)), "InvalidShape"),
    ("verify_drafts", dict(draft_probs=f(5, 50)), "InvalidShape"),
    ("verify_drafts", dict(tokens=i(5)), "InvalidShape"),
    ("verify_drafts", dict(accept_u=f(5)), "InvalidShape"),
    ("verify_drafts", dict(tokens_out=i(2, 3)), "InvalidShape"),
    ("verify_drafts", dict(path_out=i(1, 3)), "InvalidShape"),
    ("verify_drafts", dict(prob_out=f(2).double()), "InvalidType"),
    ("kv_keep_path", dict(v_caches=[]), "InvalidShape"),
    ("kv_keep_path", dict(path=q(2, 3)), "InvalidType"),
    ("kv_keep_path", dict(path=i(3, 2).T), "InvalidLayout"),
    ("kv_keep_path", dict(block_tables=i(1, 4)), "InvalidShape"),
    ("kv_keep_path", dict(context_lens=i(1)), "InvalidShape"),
]


@pytest.mark.parametrize("entry", CALLS)
def test_calls_of_these_shapes_reach_the_library(entry):
    with pytest.raises(FerrisError) as e:
        getattr(context(), entry)(**CALLS[entry])
    assert e.value.kind == "InvalidConfig" and "context" in e.value.message


@pytest.mark.parametrize("entry,change,kind", REFUSED, ids=[f"{e}-{list(c)[0]}-{n}" for n, (e, c, _) in enumerate(REFUSED)])
def test_others_are_refused(entry, change, kind):
    with pytest.raises(FerrisError) as e:
        getattr(context(), entry)(**dict(CALLS[entry], **change))
    assert e.value.kind == kind
    assert kind == "InvalidConfig" or list(change)[0] in e.value.message or entry in e.value.message
