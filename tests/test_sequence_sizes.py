"""Sizes beyond the sequence operators' range are refused before anything is allocated or called: the C descriptors hold 32
bits of each, which of 2^32 + 8 slots leaves 8. (Tensors of the meta device, which have sizes and no memory.)"""
import pytest
import torch

import channelestimationtransformer_amd as cet
from channelestimationtransformer_amd import ops

BIG = (1 << 32) + 8
empty = torch.empty


def tensor(*shape, dtype=torch.float32):
    return empty(shape, dtype=dtype, device="meta")


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    def not_reached(*args, **kwargs):
        raise AssertionError("allocated, or the library called")
    monkeypatch.setattr(ops, "_dev_check", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(ops._cabi, "lib", not_reached)
    monkeypatch.setattr(torch.Tensor, "new_empty", not_reached)
    monkeypatch.setattr(torch, "empty", not_reached)


@pytest.mark.parametrize("B, T, H", [(1, BIG, 1), (BIG, 1, 1), (1, 1, BIG), (1 << 16, 1, 1 << 16), (1, (1 << 30) + 1, 1)])
def test_linear_attention(B, T, H):
    q = tensor(B, T, H, 1)
    with pytest.raises(RuntimeError, match="served"):
        cet.linear_attention(q, q, q, tensor(H))


@pytest.mark.parametrize("B, H, rows", [(BIG, 1, None), (1, BIG, None), (4, 1, BIG), (4, 1, 1 << 31)])
def test_linear_attention_step(B, H, rows):
    q, slots = tensor(B, H, 1), None if rows is None else tensor(B, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="served"):
        cet.linear_attention_step(q, q, q, tensor(H), tensor(rows or B, H, 1, 1), slots=slots, inplace=True)


@pytest.mark.parametrize("B, T, Hq, Hk", [(1, BIG, 1, 1), (BIG, 1, 1, 1), (1, 1, BIG, 1), (1, 1, 1, BIG), (1 << 16, 1 << 16, 1, 1)])
def test_rotary(B, T, Hq, Hk):
    with pytest.raises(RuntimeError, match="served"):
        cet.rotary(tensor(B, T, Hq, 2), tensor(B, T, Hk, 2), tensor(T, dtype=torch.int64), tensor(1, dtype=torch.float64))


@pytest.mark.parametrize("N, D, F", [(BIG, 1, 1), (1, BIG, 1), (1, 1, BIG)])
def test_gated_linear(N, D, F):
    with pytest.raises(RuntimeError, match="served"):
        cet.gated_linear(tensor(N, D), tensor(F, D), tensor(F, D))
