"""Prepared plans run from a thread that has made no CUDA call before: the answers of the thread that prepared them."""
import threading

import numpy as np
import pytest

from computelibrary_b200 import capi
from helpers import q8_uniform

pytestmark = pytest.mark.gpu


def in_a_new_thread(call):
    failed = []

    def run():
        try:
            call()
        except BaseException as e:
            failed.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert not failed, failed


@pytest.mark.parametrize("M,N,K", [(16, 64, 256), (512, 256, 512), (2560, 2048, 512)])
def test_product(ctx, M, N, K):
    import torch
    r = np.random.default_rng(M)
    a, b = (torch.from_numpy(q8_uniform(r, s, np.uint8)).cuda() for s in ((M, K), (K, N)))
    desc, keep = capi.make_gemm_desc(M, N, K, capi.U8, capi.U8, capi.S32, -3, -7, stage=capi.STAGE_NONE)
    plan = capi.GemmPlan(ctx, desc, keep)
    plan.prepare(b)
    want, got = (torch.zeros((M, N), dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    in_a_new_thread(lambda: plan.run(a, b, None, got))
    plan.run(a, b, None, want)
    ctx.sync()
    plan.close()
    assert torch.equal(got, want) and want.any()


@pytest.mark.parametrize("C_,k", [(64, 1), (128, 3), (48, 3)])
def test_convolution(ctx, C_, k):
    import torch
    r = np.random.default_rng(C_)
    B, H, OFM = 2, 14, 128
    src, w = q8_uniform(r, (B, H, H, C_), np.uint8), q8_uniform(r, (OFM, k, k, C_), np.uint8)
    m, s = capi.calculate_quantized_multiplier(0.0005)
    desc, keep = capi.make_conv_desc(B, H, H, C_, OFM, k, k, (1, 1), (k // 2,) * 4, (1, 1), capi.U8, capi.U8, 5, 9, multiplier=m, shift=s,
                                     dst_zp=3, min_bound=0, max_bound=255, has_bias=False)
    plan = capi.ConvPlan(ctx, desc, keep)
    plan.prepare(torch.from_numpy(w).cuda())
    x = torch.from_numpy(src).cuda()
    want, got = (torch.zeros((B, H, H, OFM), dtype=torch.uint8, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    in_a_new_thread(lambda: plan.run(x, None, got))
    plan.run(x, None, want)
    ctx.sync()
    plan.close()
    assert torch.equal(got, want) and want.any()
