"""CPU: the workspace of the embedding backward with ordered norm gradients follows the grid, and a smaller one is refused."""
import ctypes


def test_workspace_query_and_refusal():
    from scoreperformer_amd import build, lib
    build.build()
    handle = lib.load()
    q = lambda T, D: handle.spn_embed_bwd_det_workspace_floats(T, D)
    old = lib.get_tuning("embed_stats_blocks")
    try:
        lib.set_tuning("embed_stats_blocks", 2048)
        assert q(0, 8) == 0 and q(4, 1536) == 8                                  # one block: nothing to add up
        assert q(128, 1536) == 2 * 128 + 2 * 32 * 1536                           # 4 rows a block at least
        assert q(131072, 1536) == 2 * 131072 + 2 * 2048 * 1536
        lib.set_tuning("embed_stats_blocks", 8)
        assert q(128, 1536) == 2 * 128 + 2 * 8 * 1536
        assert q(2 ** 31 - 1, 2048) > 2 ** 32
    finally:
        lib.set_tuning("embed_stats_blocks", old)
    buf = (ctypes.c_float * 4096)()
    at, one = ctypes.addressof(buf), (ctypes.c_int * 1)(8)
    ptrs = (ctypes.c_void_p * 1)(at)
    p, i, l = ctypes.c_void_p, ctypes.c_int, ctypes.c_long
    need = q(128, 8)

    def call(floats, ws=at, T=128):
        return handle.spn_embed_bwd_det(i(1), ptrs, ptrs, one, one, p(at), l(0), l(1), i(T), p(at), l(8), p(at), p(at), p(at), p(at), p(at), p(ws), l(floats), i(T),
                                        i(0), p(0))

    for bad in (lambda: call(need - 1), lambda: call(need, ws=0), lambda: call(need, T=0), lambda: call(2 * 128)):
        assert bad() != 0 and b"spn_embed_bwd" in handle.spn_last_error()
