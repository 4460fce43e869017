"""Routing and combination at the ends of the sizes they accept, on the B200 (routing: some 60 GB)."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200.ops.experts import (  # noqa: E402
    combine_experts, combine_experts_backward, route_experts, route_experts_backward)


def test_routing_of_as_many_tokens_as_fit():
    # Two experts, one taken: every token's table entries, weight and gradient, part by part.  A
    # weight is 1 / (1 + exp(-d)) of FP32 operations (5e-6 as in the smaller tests), the gradient
    # is rounded to BF16 on top of that.
    T, part = 2**31 - 1, 2**26
    logits = torch.empty(T, 2, device="cuda", dtype=torch.bfloat16)
    grad = torch.empty(T, 1, device="cuda")
    for a in range(0, T, part):
        logits[a : a + part].normal_()
        grad[a : a + part].normal_()
    r = route_experts(logits, 1, renormalize=False)
    dl = route_experts_backward(logits, r, grad, renormalize=False)
    seconds = sum(int((logits[a : a + part, 1] > logits[a : a + part, 0]).sum()) for a in range(0, T, part))
    assert r.offsets.tolist() == [0, T - seconds, T]
    at = [0, T - seconds]
    for a in range(0, T, part):
        l, g = logits[a : a + part].double(), grad[a : a + part, 0].double()
        second = l[:, 1] > l[:, 0]
        assert torch.equal(r.experts[a : a + part, 0], second.int())
        for e in (0, 1):
            taken = second if e else ~second
            n = int(taken.sum())
            want = torch.arange(at[e], at[e] + n, device="cuda")
            assert torch.equal(r.positions[a : a + part, 0][taken].long(), want)
            tokens = torch.nonzero(taken)[:, 0] + a
            assert torch.equal(r.rows[at[e] : at[e] + n].long(), tokens)
            at[e] += n
        w = torch.sigmoid((l[:, 1] - l[:, 0]).abs())
        assert ((r.weights[a : a + part, 0] - w).abs() <= 5e-6 * w).all()
        slope = w * (1 - w) * g
        want = torch.where(second[:, None], torch.stack((-slope, slope), 1), torch.stack((slope, -slope), 1))
        far = (dl[a : a + part].double() - want).abs() - 2.0**-8 * want.abs()
        assert (far <= 2e-5 * (w * g).abs()[:, None]).all()
    assert at == [T - seconds, T]
    del logits, grad, r, dl
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 65535 * 1024 + 1037), (torch.float32, 65535 * 512 + 8), (torch.float16, 2**27 + 64)])
def test_combination_of_rows_wider_than_one_grid(dtype, width):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = route_experts(torch.randn(2, 3, generator=g, device="cuda"), 2)
    y = torch.empty(4, width, device="cuda", dtype=dtype).normal_(generator=g)
    out = combine_experts(y, r.weights, r.positions)
    unit = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    grad_y, _ = combine_experts_backward(out, y, r.weights, r.positions)
    for a in range(0, width, 2**24):
        part = slice(a, a + 2**24)
        for t in range(2):
            terms = [r.weights[t, j].double() * y[int(r.positions[t, j]), part].double() for j in range(2)]
            far = (out[t, part].double() - terms[0] - terms[1]).abs()
            assert (far <= (2 * 2.0**-24 + unit) * (terms[0].abs() + terms[1].abs()) + 2.0**-24).all()
            for j in range(2):
                want = r.weights[t, j].double() * out[t, part].double()
                assert ((grad_y[int(r.positions[t, j]), part].double() - want).abs() <= unit * want.abs() + 2.0**-24).all()
