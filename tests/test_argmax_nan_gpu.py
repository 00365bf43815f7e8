"""Greedy tokens of logits that are NaN: always rows of the embedding."""

import pytest
import torch

from torchnative_b200 import _native as N

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("vocab", [999, 2048])
def test_rows_with_nan_have_a_token(cuda_device, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((4, vocab), generator=g).to(BF).to(cuda_device)
    embed = torch.randn((vocab, 64), generator=g).to(BF).to(cuda_device)
    logits[0] = float("nan")
    logits[1] = -float("inf")
    logits[2, ::3] = float("nan")
    tokens = torch.full((4,), 5, dtype=torch.int32, device=cuda_device)
    h = torch.zeros((4, 64), dtype=BF, device=cuda_device)
    N.check(N.lib().tn_llama_argmax_embed(logits.data_ptr(), 4, vocab, tokens.data_ptr(), embed.data_ptr(), 64, h.data_ptr(),
                                          None, torch.cuda.current_stream().cuda_stream))
    want = logits.float().nan_to_num(-float("inf"), neginf=-float("inf")).argmax(-1)
    assert want[:2].tolist() == [0, 0]
    assert torch.equal(tokens, want.to(torch.int32)) and torch.equal(h, embed[want])


def test_the_persistent_kernel_too(cuda_device):
    from torchnative_b200.llama_decode import LLAMA3_8B, Q4LlamaDecoder

    dec = Q4LlamaDecoder(LLAMA3_8B, batch=1, capacity=64, device=cuda_device, seed=3, layers=1, mega=True)
    dec.lm_head.view(-1, 18)[:, 1] = 0x7e  # every scale NaN
    dec.fill_prompt_cache(40)
    dec.start(torch.tensor([17], device=cuda_device))
    dec.step()
    assert dec.logits.isnan().all() and dec.tokens.tolist() == [0]
    N.device_status()
    dec.close()
