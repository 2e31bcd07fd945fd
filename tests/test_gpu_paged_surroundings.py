"""GPU: the operators on a paged cache and rotary positions among what programs do around them: host threads, activation
checkpoints, graphs that share a pool, compiled calls of changing sizes, transforms that cannot handle writes."""
import functools
import threading

import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, make_cache
from test_gpu_dispatch import setup, step
from test_gpu_paged_cache import freq, tokens

pytestmark = pytest.mark.gpu


def some_args():
    return [*setup(), torch.zeros(2, 40, device="cuda"), freq(512)]


@pytest.mark.parametrize("own_stream", [False, True])
def test_host_threads(own_stream):
    base = some_args()
    want = step(*[a.clone() for a in base])
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            for _ in range(40):
                got = step(*[a.clone() for a in base])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert_status_ok()


def test_graphs_that_share_a_pool():
    base = some_args()
    want = step(*[a.clone() for a in base])
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for _ in range(2):
        args = [a.clone() for a in base]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = step(*args)
        graphs.append((graph, out, args))
    for graph, out, args in graphs * 2:  # one after the other, as a shared pool asks for
        for a, b in zip(args, base):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert_status_ok()


def test_activation_checkpoints():
    from torch.utils.checkpoint import checkpoint, create_selective_checkpoint_contexts
    from splitd_flash_attn import split_flash_attn_func, split_rotary_func

    qkv = [tokens((2, 64), h, torch.bfloat16, h + i) for i, h in enumerate((8, 2, 2))]
    dy, pos, f = tokens((2, 64), 8, torch.bfloat16, 4), torch.arange(64, device="cuda"), freq(512)

    def fn(q, k, v):
        qr, kr = split_rotary_func(q, k, pos, f)
        return split_flash_attn_func(qr, kr, v, causal=True)

    def grads(run):
        leaves = [t.clone().requires_grad_() for t in qkv]
        return torch.autograd.grad(run(*leaves), leaves, dy)

    want = grads(fn)
    ops = torch.ops.splitd_flash_attn
    for saved in (None, [], [ops.rotary.default], [ops.fwd.default]):
        how = {} if saved is None else {"context_fn": functools.partial(create_selective_checkpoint_contexts, saved)}
        got = grads(lambda *x: checkpoint(fn, *x, use_reentrant=False, **how))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), saved
    assert_status_ok()


def test_compiled_calls_of_changing_sizes():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_evict_func

    def fn(q, k, v, table, seqlens, w, new, keep):
        out = split_flash_attn_paged_func(q, k, v, table, seqlens, causal=True, key_weights=w)
        return (out, *split_paged_evict_func(k, v, table, seqlens, w, new, keep, 1, 1, weights_len=keep + 7))

    compiled = torch.compile(fn, dynamic=True, fullgraph=True)
    for lens, keep in (([40, 21], 24), ([40, 21, 70], 24), ([10] * 5, 9), ([90, 3], 33)):
        B, need = len(lens), -(-keep // 16)
        k, v, table, seqlens, free = make_cache(lens, 16, 2, torch.bfloat16, B, spare=need * B, fill=0.0)
        q, new = tokens((B, 1), 8, torch.bfloat16, B), free.view(B, need)
        results = []
        for run in (fn, compiled):
            w = torch.zeros(B, 100, device="cuda")
            results.append((*run(q, k.clone(), v.clone(), table, seqlens, w, new, keep), w))
        assert all(torch.equal(a, b) for a, b in zip(*results))
    assert_status_ok()


def test_transforms_refuse_writes():
    base = some_args()
    kept = [a.clone() for a in base]
    with pytest.raises(RuntimeError):
        torch.func.functionalize(step)(*base)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda q: step(q, *base[1:]))(torch.stack((base[0], base[0])))
    assert all(torch.equal(a, b) for a, b in zip(base, kept)) and base[0].shape[-1] == D
    assert_status_ok()
