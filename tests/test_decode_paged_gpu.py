"""The Q4_0 decode engine over the paged 4-bit cache: each layer's attention block on its own inputs, every sequence at
a length of its own, idle sequences, and the step as one graph."""

import pytest
import torch

from tests.kv_q4_ref import attention
from torchnative_b200 import _native as N
from torchnative_b200 import kv_cache as kv

pytestmark = pytest.mark.gpu


def small(batch, device, **kw):
    from torchnative_b200.llama_decode import LlamaShape, Q4LlamaDecoder

    shape = LlamaShape(hidden=512, inter=1024, heads=8, kv_heads=2, head_dim=64, vocab=2048, layers=2, rope_theta=10000.0)
    return Q4LlamaDecoder(shape, batch=batch, capacity=80, device=device, seed=12, kv_cache="q4_0", page_size=16, **kw)


def tokens(batch, device):
    return (torch.arange(batch, dtype=torch.int32, device=device) * 131 + 7) % 2048


@pytest.mark.parametrize("lengths", [[30], [33, 0, 16], [30, 1, 64, 0, 47, 16], [7 + 3 * i for i in range(18)]])
def test_the_last_layers_attention_on_its_own_inputs(cuda_device, lengths):
    b = len(lengths)
    dec = small(b, cuda_device)
    dec.fill_prompt_cache(lengths)
    dec.start(tokens(b, cuda_device))
    before = dec.paged.pools[1].clone()
    dec.step()
    dec.paged.check()
    c = dec.paged
    after = [n + 1 if n else 0 for n in lengths]
    assert c.lengths.tolist() == after
    q, k, v = dec.qkv_out.unflatten(1, (-1, 64)).split([8, 2, 2], 1)
    at = torch.tensor([max(n, 0) for n in lengths], device=cuda_device)
    cos, sin = dec.rope[at].float()[:, None].chunk(2, -1)

    def rotate(x):
        a, e = x.float().chunk(2, -1)
        return torch.cat((a * cos - e * sin, e * cos + a * sin), -1).to(x.dtype)

    q, k = rotate(q), rotate(k)
    slots = c.page_table.gather(1, (at // 16)[:, None])[:, 0].long() * 16 + at % 16
    kv.kv_q4_append(k.contiguous(), v.contiguous(), before, torch.where(c.lengths > 0, slots, -1))
    assert torch.equal(before, c.pools[1])
    want, _, bound, _ = attention(q, c.pools[1], c.page_table, c.lengths, 16)
    got = dec.attn.view(b, 8, 64).double().cpu()
    assert ((got - want).abs() <= bound).all()
    assert all((got[i] == 0).all() for i, n in enumerate(lengths) if n == 0)


@pytest.mark.parametrize("batch", [1, 3, 6])
def test_the_step_replays_as_one_graph(cuda_device, batch):
    dec = small(batch, cuda_device)
    lengths = [30 + 5 * i for i in range(batch)]
    first = tokens(batch, cuda_device)

    def seed():
        dec.fill_prompt_cache(lengths)
        dec.start(first)

    seed()
    eager = []
    for _ in range(20):
        dec.step()
        eager.append(dec.tokens.tolist())
    dec.paged.check()
    seed()
    g = dec.capture()
    seed()
    replay = []
    for _ in range(20):
        g.replay()
        replay.append(dec.tokens.tolist())
    dec.paged.check()
    assert replay == eager
    assert dec.paged.lengths.tolist() == [n + 20 for n in lengths]


def test_sequences_do_not_see_each_other(cuda_device):
    """A sequence's tokens are those it has when the others have other lengths, or none."""
    dec = small(3, cuda_device)
    runs = []
    for lengths in ([30, 44, 9], [30, 0, 0], [30, 1, 60]):
        dec.fill_prompt_cache(lengths)
        dec.start(tokens(3, cuda_device))
        runs.append([])
        for _ in range(5):
            dec.step()
            runs[-1].append(int(dec.tokens[0]))
        dec.paged.check()
    assert runs[0] == runs[1] == runs[2]


def test_a_full_cache_is_reported(cuda_device):
    dec = small(2, cuda_device)
    dec.fill_prompt_cache([80, 20])
    dec.start(tokens(2, cuda_device))
    dec.step()
    with pytest.raises(RuntimeError, match="length"):
        dec.paged.check()
    assert dec.paged.lengths.tolist() == [80, 20]


def test_refusals(cuda_device):
    with pytest.raises(ValueError, match="kv_cache"):
        from torchnative_b200.llama_decode import LlamaShape, Q4LlamaDecoder

        Q4LlamaDecoder(LlamaShape(512, 1024, 8, 2, 64, 2048, 1, 1e4), 1, 16, cuda_device, kv_cache="q8_0")
    with pytest.raises(NotImplementedError, match="persistent"):
        small(1, cuda_device, mega=True)
    dec = small(2, cuda_device)
    for lengths in ([0, 0], [81, 3], [3], [5, -1]):
        with pytest.raises(ValueError, match="lengths"):
            dec.fill_prompt_cache(lengths)
    N.device_status()
