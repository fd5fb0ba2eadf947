"""Step operators whose launches would pass HIP's 2^32 lanes are refused before any of them runs; checked
without a GPU, on addresses that are never touched."""
import ctypes

P = ctypes.c_void_p(4096)


def test_embed_grad_past_a_launch(pkg):
    L, big = pkg._lib.lib(), pkg._lib.EC_ERANGE

    def call(n, vocab, hidden, kind=1, gkind=0):
        need = L.ec_embed_grad_workspace(n, vocab, hidden)
        return L.ec_embed_grad(P, 8, n, P, kind, hidden, vocab, hidden, 0, 1.0, P, gkind, hidden, 0, P, need, None)

    assert call(1 << 26, 1000, 1 << 15) == big               # the sums: 2^26 workgroups of 128 lanes
    assert call((1 << 31) - 1, 1000, 8) == big               # 2^25 of them, and the zeros
    assert call(1 << 30, 1000, 1 << 13, kind=0) == big
    assert call(16, (1 << 31) - 1, 1 << 14) == big           # the zeros beside the small sort's 1024 lanes
    assert call(1 << 14, (1 << 31) - 1, 1 << 14) == big      # beside the large one's 512
