"""The operators from several host threads at once, each on a stream of its own."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_several_threads():
    from rbruck_alltoallv_b200.ops.moe import linear_int8, moe_few_tokens, quantize_weight_int8
    from rbruck_alltoallv_b200.ops.norm import block_norm
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)

    def rand(*n, dtype=torch.bfloat16):
        return torch.randn(*n, device="cuda", generator=gen).to(dtype)

    w13, w2, (q, s), w = rand(6, 320, 256), rand(6, 256, 160), quantize_weight_int8(rand(512, 256)), rand(256)
    inputs = [(rand(T, 256), rand(T, 6, dtype=torch.float32), rand(T, 256, dtype=torch.float32)) for T in (1, 7, 20, 60)]
    d = [rand(*x.shape, dtype=torch.float32) for x, _, _ in inputs]

    def work(i):
        x, logits, res = inputs[i]
        y = moe_few_tokens(x, logits, w13, w2)
        z = y.detach().requires_grad_()
        out, u = block_norm(res, z, w, pre_weight=w)
        g, = torch.autograd.grad((out, u), (z,), (d[i], d[i].to(torch.bfloat16)))
        return y, linear_int8(u.detach(), q, s), g

    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got, wrong = [[] for _ in range(4)], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i].append(work(i))
            stream.synchronize()
        except Exception as e:                           # the thread's failure is the test's
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for i in range(4):
        assert len(got[i]) == 20
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))
