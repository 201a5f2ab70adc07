"""A wait that runs out inside an optimiser's step: the weight is left alone, the call reports it, and the device goes on working."""
import pytest

pytestmark = pytest.mark.gpu


# one CTA; clusters of 2 and 8; the chain on single SMs and on pairs, with cut tiles and with more tiles than CTAs
@pytest.mark.parametrize("shape, pair", [((20, 30), 0), ((100, 200), 0), ((96, 1500), 0), ((1500, 96), 0), ((300, 400), 2), ((300, 400), 1), ((1500, 2100), 2), ((1500, 2100), 1)],
                         ids=str)
def test_nothing_is_stored_after_a_wait_gave_up(cake, shape, pair):
    import ctypes
    import time
    import torch
    torch.manual_seed(shape[0])
    W, G, M = (torch.randn(shape, device="cuda") for _ in range(3))
    keep = W.clone()
    cake.set_option("pair", pair)
    try:
        n = cake.lib().cakeb200_orthogonalize_workspace(shape[0], shape[1], 1, 0)
        buf = torch.empty(n + 1024, dtype=torch.uint8, device="cuda")
        at = (buf.data_ptr() + 1023) & ~1023
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        rc = cake.lib().cakeb200_selftest_orthogonalize_wait(*(ctypes.c_void_p(t.data_ptr()) for t in (W, G, M)), shape[0], shape[1], ctypes.c_void_p(at), n,
                                                             ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        waited = time.perf_counter() - t0
        assert rc == -4, (rc, cake.lib().cakeb200_last_error())  # CAKEB200_ERR_DEVICE_TIMEOUT
        assert torch.equal(W, keep)
        assert torch.equal(M, G)  # without momentum
        assert 1.5 < waited < 9, waited
        # the next step, in the same workspace, is an ordinary one
        rc = cake.lib().cakeb200_muon_step(W.data_ptr(), shape[1], 0, G.data_ptr(), shape[1], 0, M.data_ptr(), shape[1], *shape, 1.0, 0.0, 0, 0.0, 1.0, 5, 3.4445,
                                           -4.7750, 2.0315, 1e-7, at, n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        want = keep.double() - cake.cake_orthogonalize(G).double()
        assert bool(((W.double() - want).abs() <= 2.0 ** -23 * (want.abs() + 2)).all())
    finally:
        cake.set_option("pair", 0)
