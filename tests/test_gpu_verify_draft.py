"""verify_draft_ against its definition in 64 bits: counts and tokens exactly."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


def check(p, q, x, u, lens=None):
    B, N = x.shape
    acc, tok = ti.verify_draft(BE, x, p, q, u, lens)
    acc, tok = acc.cpu().numpy(), tok.cpu().numpy()
    ph, qh = p.float().cpu().numpy(), None if q is None else q.float().cpu().numpy()
    xh, uh = x.cpu().numpy(), u.cpu().numpy()
    for b in range(B):
        n = N if lens is None else int(lens[b])
        a, t = ref.verify(xh[b], ph[b], None if q is None else qh[b], uh[b], n)
        assert acc[b] == a and tok[b].tolist() == t, f"sequence {b}"
    return acc, tok


def inputs(B, N, V, dtype=torch.float32, seed=0, noise=0.7, given=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((B, N + 1, V), generator=g, device="cuda") * 2
    p = torch.softmax(logits, 2)
    q = torch.softmax(logits[:, :N] + noise * torch.randn((B, N, V), generator=g, device="cuda"), 2)
    x = torch.multinomial(q.reshape(B * N, V), 1, generator=g).reshape(B, N).to(torch.int32) if N else \
        torch.zeros((B, 0), dtype=torch.int32, device="cuda")
    u = torch.rand((B, N + 1), generator=g, device="cuda")
    return p.to(dtype), q.to(dtype) if given else None, x, u


@pytest.mark.parametrize("V", [1, 2, 17, 4095, 4096, 4097, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [True, False])
def test_vocabularies(gpu, V, dtype, given):
    """Rows of odd lengths (no row but the first is aligned), one to many work-groups a row."""
    check(*inputs(9, 4, V, dtype, V, given=given))


@pytest.mark.parametrize("N", [0, 1, 3, 16, 63, 64, 65, 130])
def test_drafts(gpu, N):
    p, q, x, u = inputs(5, N, 300, seed=N, noise=0.05)
    acc, _ = check(p, q, x, u)
    check(p, p[:, :N].contiguous(), x, u)                       # the same distribution: all accepted
    lens = torch.tensor([N, 0, N // 2, -4, N + 9], dtype=torch.int32, device="cuda")
    check(p, q, x, u, lens)
    if N:
        u[:, :N] = 0
        acc, _ = check(p, q, x, u)
        assert (acc == N).all()


def test_large_batch_and_vocabulary(gpu):
    check(*inputs(40, 3, 151937, seed=5))
    check(*inputs(300, 1, 1000, seed=6))


def test_uniforms_at_the_ends(gpu):
    """The first and the last token that can be drawn; values outside [0, 1) still draw one with weight."""
    p, q, x, u = inputs(6, 2, 9000, seed=7)
    p[:, :, :5] = 0
    p[:, :, -4100:] = 0
    top = np.nextafter(np.float32(1), np.float32(0))
    for last in (0.0, float(top), 1.0, 2.0, -1.0, math.inf, math.nan):
        u[:, -1] = last
        acc, tok = check(p, q, x, u) if not math.isnan(last) else (None, None)
    u[:, :2] = 1.0                                               # u q < p decides at equality too
    p2 = q[:, [0, 1, 1]].contiguous()
    acc, _ = check(p2, q, x, torch.full_like(u, 1.0))
    assert (acc == 0).all()                                     # 1 q < p is false where p = q


def test_sums_between_equal_weights(gpu):
    """Weights and uniforms that are whole multiples of a power of two: running sums meet the goal exactly,
    and the lowest token whose sum exceeds it is drawn."""
    V, B = 8192, 16
    p = torch.full((B, 1, V), 1 / V, device="cuda")
    u = torch.arange(B, device="cuda").float().reshape(B, 1) / B
    acc, tok = check(p, None, torch.zeros((B, 0), dtype=torch.int32, device="cuda"), u)
    assert tok[:, 0].tolist() == [V // B * b for b in range(B)]


def test_rejected_without_weight_left(gpu):
    """p <= q everywhere (unnormalized rows): drawn from p; rows of zeros draw nothing."""
    p, q, x, u = inputs(4, 2, 500, seed=8)
    q = torch.maximum(q, p[:, :2]) * 2
    u[:, :2] = 0.999
    check(p, q, x, u)
    p.zero_()
    acc, tok = check(p, q, x, u)
    assert (acc == 0).all() and (tok == -1).all()
    one = torch.zeros((4, 3, 500), device="cuda")
    one.scatter_(2, torch.cat([x, x[:, :1]], 1).long()[..., None], 1.0)       # all of p on the draft
    check(one, None, x, u)
    check(one, None, (x + 1) % 500, u)


def test_not_finite_and_negative_entries_have_no_weight(gpu):
    p, q, x, u = inputs(6, 2, 5000, seed=9)
    p[:, :, 100:200], p[:, :, 300], p[:, :, 400], p[:, :, 500] = math.nan, math.inf, -math.inf, -1.0
    q[:, :, 700:900], q[:, :, 1000], q[:, :, 1100] = math.nan, math.inf, -math.inf
    acc, tok = check(p, q, x, u)
    check(p, None, x, u)


def test_draft_tokens_outside_the_vocabulary(gpu):
    p, q, x, u = inputs(6, 3, 1000, seed=10)
    u[:, :3] = 0
    x[0, 0], x[1, 1], x[2, 2], x[3, 0] = -1, 1000, 2 ** 31 - 1, -2 ** 31
    acc, _ = check(p, q, x, u)
    assert acc[:4].tolist() == [0, 1, 2, 0]
    check(p, None, x, u)


def test_offsets_past_32_bits(gpu):
    """A batch whose probabilities hold more than 2^31 elements: the last sequences are read in place."""
    B, N, V = 130, 127, 131072
    p = torch.zeros((B, N + 1, V), device="cuda", dtype=torch.bfloat16)
    x = torch.zeros((B, N), dtype=torch.int32, device="cuda")
    p[:, :, 77] = 1.0
    x[:] = 77
    u = torch.full((B, N + 1), 0.5, device="cuda")
    lens = torch.randint(0, N + 1, (B,), device="cuda", dtype=torch.int32)
    lens[-1] = N
    p[-1, N, 77], p[-1, N, V - 1] = 0.0, 1.0
    acc, tok = ti.verify_draft(BE, x, p, None, u, lens)
    assert torch.equal(acc, lens)
    assert tok[-1, N].item() == V - 1 and tok[-2, lens[-2]].item() == 77
    assert (tok[-1, :N] == 77).all() and (tok[0, lens[0] + 1:] == -1).all()


def test_refusals(gpu):
    p, q, x, u = inputs(2, 2, 100)
    acc, tok = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty((2, 3), dtype=torch.int32, device="cuda")
    ws = ti.verify_draft_workspace(BE, p)

    def refused(*a):
        with pytest.raises(ti.ArgumentError):
            ti.verify_draft_(BE, *a)

    refused(acc, tok, None, x, p, q, u)
    refused(acc, tok, ws[:16], x, p, q, u)
    refused(acc, tok, ws, x.long(), p, q, u)
    refused(acc, tok, ws, x, p.half(), q.half(), u)
    refused(acc, tok, ws, x, p, q.bfloat16(), u)
    refused(acc, tok, ws, x, p, q[:, :1].contiguous(), u)
    refused(acc, tok, ws, x, p, q, u[:, :2].contiguous())
    refused(acc, tok, ws, x, p, q, u.double())
    refused(acc[:1], tok, ws, x, p, q, u)
    refused(acc, tok[:, :2].contiguous(), ws, x, p, q, u)
    refused(acc, tok, ws, x, p, q, u, torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused(acc, tok, ws, x, p[:, :, ::2], q[:, :, ::2], u)
    refused(acc, tok, ws, x.cpu(), p, q, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [True, False])
def test_uniforms_that_are_nan(gpu, dtype, given):
    """A last uniform of NaN exceeds nothing: the last token with weight; one of a draft's accepts nothing."""
    p, q, x, u = inputs(6, 2, 9000, dtype, seed=11, given=given)
    p[:, :, :5] = 0
    p[:, :, -4100:] = 0
    u[:, -1] = math.nan
    acc, tok = check(p, q, x, u)
    u[:3, 0] = math.nan
    acc, tok = check(p, q, x, u)
    assert (acc[:3] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tensors_aligned_to_their_elements_only(gpu, dtype):
    """Rows that begin one element behind an aligned address."""
    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        flat[1:] = x.reshape(-1)
        return flat[1:].view(x.shape)

    check(*(shifted(t) for t in inputs(7, 3, 5000, dtype, seed=12)))
