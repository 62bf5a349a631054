"""The walk for wait states behind matrix instructions (CPU)."""
import mfma_waits


def test_the_walk_asks_for_every_wait_state(tmp_path):
    """passes + 4 on this part: 8 behind a 16x16x32 product, 12 behind a 32x32x16 one, and not one fewer"""
    text = "f:\n\tv_mfma_f32_%s_bf16 a[0:3], v[0:3], v[4:7], a[0:3]\n\ts_nop 7\n%s\tv_accvgpr_read_b32 v9, a3\n\ts_endpgm\n.Lfunc_end0:\n"
    p = tmp_path / "f.s"
    for shape, states in (("16x16x32", 8), ("32x32x16", 12)):
        for more in range(-1, 2):
            wait = states + more
            body = text % (shape, "\ts_nop %d\n" % (wait - 9) if wait > 8 else "")
            if wait < 8:
                body = body.replace("s_nop 7", "s_nop %d" % (wait - 1))
            p.write_text(body)
            assert len(mfma_waits.audit(str(p))["f"]) == (1 if more < 0 else 0), (shape, wait)
