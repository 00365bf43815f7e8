"""The tensor-parallel decode steps over the paged 4-bit cache, on one GPU: both ranks of a group of two as threads of
this process, their exchanges done by the host between launches (it waits for a rank's stream, then copies), so that no
kernel waits for another's. What the exchange kernels themselves do is tested with a GPU a rank; here it is what each rank
computes on its own heads, columns and Q8_0 rows, and how many launches that takes."""

import ctypes
import threading

import pytest
import torch

from tests.test_decode_paged_gpu import tokens
from torchnative_b200 import _native as N
from torchnative_b200 import tp as tpm
from torchnative_b200.llama_decode import LlamaShape, Q4LlamaDecoder

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
WORLD, PAGE, CAP = 2, 16, 96


class Host:
    """What the ranks' threads share. Without one (`None`) an exchange is only counted."""

    def __init__(self):
        self.gate, self.given = threading.Barrier(WORLD, timeout=120), [None] * WORLD

    def exchange(self, rank, mine):
        torch.cuda.current_stream().synchronize()
        self.given[rank] = mine.clone()
        torch.cuda.current_stream().synchronize()
        self.gate.wait()
        all_ranks = [x.clone() for x in self.given]
        torch.cuda.current_stream().synchronize()
        self.gate.wait()
        return all_ranks


class Group:
    def __init__(self, rank, host):
        self.rank, self.world, self.group, self.host = rank, WORLD, None, host

    def all_gather(self, out, inp):
        if self.host is not None:
            out.view(WORLD, -1).copy_(torch.stack(self.host.exchange(self.rank, inp.reshape(-1))))


class Link:
    def __init__(self, kind, off=0):
        self.kind, self.off = kind, off


class Exchange:
    """PeerExchange with the host in the place of peer memory."""

    def __init__(self, tp, nbytes, device):
        self.tp, self.dev, self.buffers, self.launches = tp, torch.device(device), [], 0

    def buffer(self, rows, cols, dtype=BF):
        self.buffers.append(torch.zeros((rows, cols), dtype=dtype, device=self.dev))
        return self.buffers[-1], len(self.buffers) - 1

    def reserve(self, nbytes):
        return 0

    def gather(self, local, off):
        if self.tp.host is not None:
            self.buffers[off].copy_(torch.cat(self.tp.host.exchange(self.tp.rank, local.view(local.shape[0], -1)), 1))

    def allgather(self, local, off, full_cols, slot, stream):
        assert self.buffers[off].shape[1] == full_cols == WORLD * local.shape[1]
        self.launches += 1
        self.gather(local, off)

    def reduce_link(self, slot, partial_off, cols):
        return Link("reduce")

    def link(self, slot=-1, dst_off=0, full_cols=0, wait_slot=-1):
        return Link("gather", dst_off) if slot >= 0 else Link("wait")

    def step_end(self, stream):
        self.launches += 1

    def close(self):
        pass


class Rank(Q4LlamaDecoder):
    """A decoder whose linked linears run unlinked, the host doing the rest."""

    def _after(self, y, link):
        if link is None or link.kind == "wait":
            return
        if link.kind == "gather":
            self.xchg.gather(y, link.off)
        elif self.tp.host is not None:
            y.copy_(sum(x.float() for x in self.tp.host.exchange(self.tp.rank, y)).to(y.dtype))

    def _linear(self, w, y, n, k, stream, flags=0, link=None):
        if self.watch is not None and any(w is lw["o"] for lw in self.layers):
            self.watch(self, k)
        super()._linear(w, y, n, k, stream, flags)
        self._after(y, link)

    def _fused_linear(self, mode, x, x_stride, delta, h_out, norm_w, w, y, n, k, stream, flags=0, link=None, q8=False):
        super()._fused_linear(mode, x, x_stride, delta, h_out, norm_w, w, y, n, k, stream, flags, None, q8)
        self._after(y, link)

    watch = None


def shape(inter):
    return LlamaShape(hidden=512, inter=inter, heads=8, kv_heads=4, head_dim=64, vocab=2048, layers=2, rope_theta=10000.0)


def rank_decoder(rank, host, device, batch, inter, exchange, plan, **kw):
    return Rank(shape(inter), batch, CAP, device, seed=12, tp=Group(rank, host), exchange=exchange, tp_plan=plan,
                kv_cache="q4_0", page_size=PAGE, **kw)


def planar(x):
    rows, k = x.shape
    out = (torch.empty((rows, k), dtype=torch.int8, device=x.device), torch.empty((rows, k // 32), device=x.device),
           torch.empty((rows, k // 32), device=x.device))
    N.check(N.lib().tn_q8_0_quantize_planar(x.data_ptr(), N.TN_BF16, k, out[0].data_ptr(), k, out[1].data_ptr(),
                                            out[2].data_ptr(), rows, k, torch.cuda.current_stream().cuda_stream))
    return out


PLANS = [("nccl", "colwise"), ("p2p", "colwise"), ("p2p", "rowwise")]


@pytest.mark.parametrize("batch, inter", [(1, 1024), (3, 1024), (4, 5120), (6, 1024), (18, 1024)])
@pytest.mark.parametrize("exchange, plan", PLANS)
def test_both_ranks_steps(cuda_device, monkeypatch, batch, inter, exchange, plan):
    """Under the colwise plan each rank's pools and tokens are the one-GPU decoder's; under both plans what o_proj takes is
    the planar Q8_0 of the attention output, of the rank's own heads where it is row-parallel."""
    monkeypatch.setattr(tpm, "PeerExchange", Exchange)
    lengths = [30 + 3 * i for i in range(batch)]
    if batch > 2:
        lengths[1] = 0
    one = Q4LlamaDecoder(shape(inter), batch, CAP, cuda_device, seed=12, kv_cache="q4_0", page_size=PAGE)
    one.fill_prompt_cache(lengths)
    one.start(tokens(batch, cuda_device))
    want = []
    for _ in range(3):
        one.step()
        want.append((one.tokens.clone(), [p.clone() for p in one.paged.pools], one.paged.lengths.clone()))
    one.paged.check()
    host, got, failed = Host(), [[] for _ in range(WORLD)], []

    def watch(dec, k):
        x = (dec.attn_l if dec.rowwise else dec.attn).reshape(batch, -1)
        assert x.shape[1] == k
        for a, b in zip(planar(x), (dec.codes, dec.scales, dec.offsets)):
            assert torch.equal(a, b.view(-1)[:a.numel()].view_as(a))

    def work(rank):
        try:
            with torch.cuda.device(cuda_device), torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                dec = rank_decoder(rank, host, cuda_device, batch, inter, exchange, plan)
                assert dec.rowwise == (plan == "rowwise" and batch <= 16)
                dec.watch = watch
                dec.fill_prompt_cache(lengths)
                dec.start(tokens(batch, cuda_device))
                for _ in range(3):
                    dec.step()
                    got[rank].append((dec.tokens.clone(), [p.clone() for p in dec.paged.pools], dec.paged.lengths.clone(),
                                      dec.rowwise, dec.hkv))
                torch.cuda.current_stream().synchronize()
                assert dec.paged.status.item() == 0
        except BaseException as e:  # noqa: BLE001 -- shown below; the other rank's wait ends
            failed.append(e)
            host.gate.abort()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(r,)) for r in range(WORLD)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]
    N.device_status()
    for rank in range(WORLD):
        for i, ((tok, pools, after), (t, ps, a, rowwise, hkv)) in enumerate(zip(want, got[rank])):
            assert torch.equal(a, after)
            mine = slice(rank * hkv, (rank + 1) * hkv)
            if rowwise:  # the host adds rounded partial rows: from layer 1 on the numbers differ in their last bits
                assert torch.equal(t, got[0][i][0])
                if i == 0:
                    assert torch.equal(ps[0], pools[0][:, mine])
            else:
                assert torch.equal(t, tok)
                assert all(torch.equal(x, y[:, mine]) for x, y in zip(ps, pools))


@pytest.mark.parametrize("batch, inter", [(1, 1024), (4, 5120), (6, 1024), (18, 1024)])
@pytest.mark.parametrize("exchange, plan", [*PLANS, (None, "colwise")])
def test_launches_of_a_step(cuda_device, monkeypatch, batch, inter, exchange, plan):
    """kernels_per_step is what a captured step holds, and the exchange's own launches."""
    monkeypatch.setattr(tpm, "PeerExchange", Exchange)
    if exchange is None:
        dec = Q4LlamaDecoder(shape(inter), batch, CAP, cuda_device, seed=12, kv_cache="q4_0", page_size=PAGE)
    else:
        dec = rank_decoder(0, None, cuda_device, batch, inter, exchange, plan)
    dec.fill_prompt_cache([20] * batch)
    dec.start(tokens(batch, cuda_device))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step()
    side.synchronize()
    if dec.xchg is not None:
        dec.xchg.launches = 0
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=side):
        dec.step()
    nodes = ctypes.c_size_t()
    count = ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes
    assert count(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    launches = nodes.value + (0 if dec.xchg is None else dec.xchg.launches)
    assert launches == dec.kernels_per_step
