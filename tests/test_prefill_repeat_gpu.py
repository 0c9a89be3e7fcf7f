"""The paged and contiguous prefill called again and again while another stream keeps HBM busy, so that
values arrive late: every call has the same bits, and the first is right."""

import math

import pytest
import torch

import oracle
from _util import bits_equal, cuda_device, stream
from test_prefill_gpu import TOL, make_paged
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch.attention import flash_attn_varlen_func, paged_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qlens,ctxs", [([512, 1024], [2048, 1024]), ([128] * 9, [256 + 128 * b for b in range(9)]),
                                        ([100] * 40, [130 + 7 * b for b in range(40)])], ids=["long", "prefix", "short"])
def test_prefill_repeats_its_bits_beside_other_traffic(qlens, ctxs):
    dev = cuda_device()
    torch.cuda.synchronize()
    capi.read_device_error(stream())
    scale = 1.0 / math.sqrt(128)
    q, kc, vc, cu, seq, table = make_paged(qlens, ctxs, 32, 8, seed=91)
    ref = oracle.paged_prefill(q, kc, vc, cu, seq, table, scale)
    qd, kd, vd, cud, seqd, tabled = (t.to(dev) for t in (q, kc, vc, cu, seq, table))
    cu_k = torch.tensor([0] + torch.tensor(ctxs).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    rows = [(int(table[b, i // 16]), i % 16) for b, n in enumerate(ctxs) for i in range(n)]
    at = torch.tensor(rows, device=dev)
    k, v = kd[at[:, 0], at[:, 1]], vd[at[:, 0], at[:, 1]]
    side, a = torch.cuda.Stream(dev), torch.empty(1 << 28, dtype=torch.uint8, device=dev)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    paged, contiguous = [], []
    for _ in range(60):
        with torch.cuda.stream(side):
            for _ in range(3):
                b.copy_(a)
        out = torch.full_like(qd, float("nan"))
        paged_prefill(out, qd, kd, vd, cud, seqd, tabled, max(qlens), scale, True)
        paged.append(out)
        contiguous.append(flash_attn_varlen_func(qd, k, v, cud, cu_k, max(qlens), softmax_scale=scale, causal=True))
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    torch.testing.assert_close(paged[0].float().cpu(), ref, rtol=TOL, atol=TOL)
    torch.testing.assert_close(contiguous[0].float().cpu(), ref, rtol=TOL, atol=TOL)
    for out in paged[1:]:
        assert bits_equal(out, paged[0])
    for out in contiguous[1:]:
        assert bits_equal(out, contiguous[0])
