"""Append, attention with weights and eviction together, as kv4_example runs them, step by step against the definition in 64 bits (tolerances as in test_gpu_kv4.py)."""
import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv4 import no_wait_ran_out  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,page,room,keep,prompt,steps", [(8, 2, 16, 96, 40, 50, 130), (4, 4, 64, 192, 127, 64, 140), (16, 1, 32, 128, 33, 90, 100)])
def test_generation_with_a_bounded_cache(heads, kv_heads, page, room, keep, prompt, steps):
    from amdgpu_rustdsl_b200 import kv4_read
    from amdgpu_rustdsl_b200.kv4_example import BoundedCache
    B, recent, first = 3, 8, 2
    layer = BoundedCache(B, kv_heads, room, keep, recent, first, page)
    g = torch.Generator().manual_seed(heads)
    evictions = 0

    def values(cache, n):
        k, v = (torch.empty(B, n, kv_heads, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kv4_read(cache, k, v)
        return k.cpu(), v.cpu()

    for step in range(steps):
        S = prompt if step == 0 else 1
        counts = [prompt, prompt // 2, 1] if step == 0 else None
        x = torch.randn(B, S, heads + 2 * kv_heads, 128, generator=g).bfloat16().cuda()
        q, k, v = x.split([heads, kv_heads, kv_heads], 2)
        out = torch.full((B, S, heads, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
        before, lengths, weights = layer.cache, layer.cache.lengths.tolist(), layer.weights[0].cpu()
        if layer.make_room(S):
            evictions += 1
            assert layer.cache is not before
            stay = R.evict(weights, lengths, keep, recent, first)
            assert layer.cache.lengths.tolist() == [min(n, keep) for n in lengths]
            (old_k, old_v), (new_k, new_v) = values(before, max(lengths)), values(layer.cache, keep)
            for b in range(B):
                for h in range(kv_heads):
                    at = torch.tensor(stay[b][h])
                    assert torch.equal(new_k[b, :len(at), h], old_k[b, at, h]) and torch.equal(new_v[b, :len(at), h], old_v[b, at, h])
                    assert torch.equal(layer.weights[0][b, h, :len(at)].cpu(), weights[b, h, at])
        weights_in = layer.weights[0].cpu()
        layer.step(q, k, v, out, None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert layer.cache.lengths.max().item() <= room
        if step % 7 not in (0, 1) and step + 1 < steps:   # (the reference takes its time)
            continue
        cache = layer.cache
        ref, _, ref_w, spread, peak, size, doubt = R.attend(q.cpu(), cache.pool.cpu(), cache.table.cpu(), cache.lengths.cpu(), True, counts, None, weights_in)
        off = 128 * 2.0 ** -24 * size + 2.0 ** -21
        got = out.cpu().double()
        allowed = 2.0 ** -9 * ref.abs() + spread * (2.0 ** -9 + 4 * off.permute(0, 2, 1)[..., None]) * 1.01 + (room * 1.5 * 2.0 ** -25 * peak)[..., None] + 1e-38
        assert ((got - ref).abs() <= allowed).all()
        live = (torch.arange(ref_w.shape[-1]) < cache.lengths.cpu()[:, None, None]).expand_as(ref_w)
        w = layer.weights[0].cpu().double()
        assert ((w - ref_w).abs() <= 2 * (128 * 2.0 ** -24 * doubt + 2.0 ** -20 * ref_w.abs()) + 1e-30)[live].all()
    assert evictions >= 1


def test_the_room_is_checked():
    from amdgpu_rustdsl_b200.kv4_example import BoundedCache
    with pytest.raises(ValueError, match="keep must be"):
        BoundedCache(1, 1, 64, 64, page=16)
    with pytest.raises(ValueError, match="keep must be"):
        BoundedCache(1, 1, 64, 20, recent=20, first=4, page=16)
    layer = BoundedCache(1, 1, 64, 40, recent=20, first=4, page=16)
    x = torch.zeros(1, 25, 1, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="24 fit"):
        layer.step(x, x, x, torch.empty_like(x))


def test_the_command_runs(capsys):
    from amdgpu_rustdsl_b200 import kv4_example
    kv4_example.main("--sequences 2 --heads 4 --kv-heads 2 --prompt 300 --chunk 100 --steps 300 --room 512 --keep 256".split())
    assert "generation, 2 sequences" in capsys.readouterr().out
