"""Positions of the wrong shape are refused before a device reads them: a consumer takes its token
count from them, and reads a row of partials and a slot, and writes a query row, for each."""
from types import SimpleNamespace

import pytest
import torch

from ferrisinfer_amd import FerrisError, kernel
from ferrisinfer_amd.bf16_decoder import Bf16Decoder, StepBatch

T = 6


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("pair_axes,positions,slots", [
    (None, (3, T), T),       # several axes to a decoder of one
    (None, (T + 1,), T),
    (None, (T - 1,), T),
    ([0, 1, 2, 0], (3, T + 1), T),
    ([0, 1, 2, 0], (T, 3), T),      # transposed
    ([0, 1, 2, 0], (3, 1, T), T),
    ([0, 1, 2, 0], (3, T), T - 1),
    (None, (T,), T - 1),
])
def test_decoder_step_refuses_positions_of_other_rows(pair_axes, positions, slots):
    dec = object.__new__(Bf16Decoder)
    dec.ctx, dec.cfg, dec.max_tokens, dec.pair_axes, dec.layers = None, {}, 64, pair_axes, [{}]
    batch = StepBatch(positions=ints(*positions), slot_mapping=torch.zeros(slots, dtype=torch.int64), num_decode=T,
                      dec_block_tables=None, dec_context_lens=None, dec_max_context=0, pf_block_tables=None,
                      pf_cu_seqlens=None, pf_context_lens=None, pf_max_query=0, last_rows=None)
    with pytest.raises(FerrisError) as e:
        dec.step(torch.zeros(T, 4), batch)
    assert e.value.kind == "InvalidShape"


@pytest.mark.parametrize("pair_axes,positions,slots", [(None, (T,), T), (None, (T,), T + 3), (None, (1, T), T),
                                                       ([0, 1, 2, 0], (3, T), T), ([0, 0, 0, 0], (T,), T)])
def test_decoder_step_takes_positions_of_its_rows(pair_axes, positions, slots):
    dec = object.__new__(Bf16Decoder)
    dec.ctx, dec.cfg, dec.max_tokens, dec.pair_axes, dec.layers = None, {}, 64, pair_axes, []
    batch = StepBatch(positions=ints(*positions), slot_mapping=torch.zeros(slots, dtype=torch.int64), num_decode=T,
                      dec_block_tables=None, dec_context_lens=None, dec_max_context=0, pf_block_tables=None,
                      pf_cu_seqlens=None, pf_context_lens=None, pf_max_query=0, last_rows=None)
    with pytest.raises(FerrisError) as e:  # the next check: a decoder without layers
        dec.step(torch.zeros(T, 4), batch)
    assert e.value.kind != "InvalidShape" and "layers" in e.value.message


def context():
    """A context without a device: what reaches the library is refused there as InvalidConfig."""
    ctx = object.__new__(kernel.Context)
    ctx.lib, ctx.handle = kernel.load(), None
    return ctx


def consume(entry, positions, slots):
    p = SimpleNamespace(data_ptr=lambda: 16)
    tail = (p, p, 32, 8, torch.zeros(slots, dtype=torch.int64), p, p, 0, 4, 16, 2, 1, 32, p)
    if entry == "qkv_rope_append":
        context().qkv_rope_append(p, 1, None, positions, *tail)
    else:
        context().qkv_norm_rope_append(p, 1, None, None, 0.0, positions, None, *tail)


@pytest.mark.parametrize("entry,shape,slots", [
    ("qkv_rope_append", (3, T), T),
    ("qkv_rope_append", (T,), T - 1),
    ("qkv_norm_rope_append", (1, T), T - 1),
    ("qkv_norm_rope_append", (T,), T - 1),
    ("qkv_norm_rope_append", (1, 1, T), T),
    ("qkv_norm_rope_append", (), T),
])
def test_consumers_refuse_more_positions_than_slots(entry, shape, slots):
    with pytest.raises(FerrisError) as e:
        consume(entry, ints(*shape), slots)
    assert e.value.kind == "InvalidShape"


@pytest.mark.parametrize("entry", ["qkv_rope_append", "qkv_norm_rope_append"])
def test_as_many_positions_as_slots_reach_the_library(entry):
    with pytest.raises(FerrisError) as e:  # no context
        consume(entry, ints(T), T)
    assert e.value.kind != "InvalidShape"
