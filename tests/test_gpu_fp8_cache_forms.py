"""Writes into 8-bit block caches at the forms that the launch picks between: fused and Float32 calls, whose full pages are
read twice, and pages of up to 1024 keys."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from test_gpu_fp8_cache import pools, rows, same
from test_gpu_fp8_cache import test_fused_inputs_are_the_ops_in_a_row as fused_is_the_ops_in_a_row
from window_ref import i32, store

BE = ti.HipBackend()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,nq,H,P,n", [(128, 4, 2, 128, 700), (128, 2, 3, 1024, 3000), (64, 4, 9, 256, 900), (64, 2, 17, 64, 2100), (128, 8, 8, 32, 5000),
                                        (128, 1, 1, 1024, 256), (64, 1, 2, 512, 257)])
def test_fused_forms(gpu, T, D, nq, H, P, n):
    fused_is_the_ops_in_a_row(gpu, T, True, D, nq, H, P, n)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,H,P,n", [(128, 8, 1024, 3000), (128, 3, 256, 2000), (64, 9, 512, 4000), (128, 17, 64, 1500), (128, 1, 16, 257)])
def test_full_pages(gpu, T, D, H, P, n):
    """Pages written whole and in parts, in order and mixed up, over what they held."""
    g = np.random.Generator(np.random.PCG64(P + n))
    pages = n // P + 3
    k, v = pools(D, P, H, pages, g)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    order = np.arange(n) + 1
    for at in (order, order + P // 2, g.permutation(pages * P)[:n] + 1):
        x, y = rows(g, n, H, D, T), rows(g, n, H, D, T)
        ti.store_kv_(BE, k, v, x.cuda(), y.cuda(), i32(at))
        store(q, scale, x.float().numpy(), y.float().numpy(), list(at))
        same(k, q, scale)
