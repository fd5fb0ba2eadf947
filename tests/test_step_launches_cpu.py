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


def test_the_sorts_memory_does_not_grow_with_the_tokens(pkg):
    """Besides 16 bytes a token and the sums' two parts for each 32 tokens: each workgroup of the sort reads all
    counts, so their number has a limit."""
    ws = pkg._lib.lib().ec_embed_grad_workspace
    for vocab in (50_304, 262_143, 1 << 30):
        sizes = [ws(n, vocab, 1) - 16 * n - 8 * (n // 32) for n in (1 << 20, 1 << 24, 1 << 30)]
        assert sizes[0] == sizes[1] == sizes[2] <= 512 * 4 * (512 + 8192), sizes
