"""Where label operators' scratch memory and codes lie, on the CPU: strides that vector loads need, and offsets that pass 32 bits.  The offsets are
those of renee_amd/csrc/mx4_layout.hpp, which the kernels take them from."""
import os
import shutil
import subprocess

import pytest

from renee_amd._lib import lib

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "renee_amd", "csrc")


@pytest.mark.parametrize("rows", [1, 3, 256, 300])
@pytest.mark.parametrize("K", [9, 300, 6000])
def test_maxima_beside_logits_are_rows_of_whole_pieces(rows, K):
    """The selection reads a row's maxima, one half for every 32 labels, in pieces of 16 bytes: each row begins on one, and the last row's
    last piece is inside the workspace."""
    h = lib()
    for L in [*range(65_473, 65_900, 7), 70_001, 131_072, 320_001, 414_001, 1_310_720, 2_812_281, (1 << 30) - 1]:
        if L < K * 64:
            continue
        d = 4096  # wide enough for every K to go by logits
        logits = (rows * -(-L // 64) * 64 * 2 + 15) // 16 * 16
        maxima = h.xfc_mx4_topk_workspace_bytes(rows, L, d, K) - logits
        blocks = -(-L // 32)
        if rows >= 32 and maxima < 0:  # by maxima alone
            continue
        if maxima == 0:  # too few blocks for them to be of use
            assert blocks < 2048 or blocks < 2 * K
            continue
        assert maxima % rows == 0 and maxima // rows % 16 == 0
        assert maxima // rows >= -(-blocks // 8) * 16


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    """The layout's functions: name, arguments -> value."""
    gxx = shutil.which("g++") or shutil.which("clang++", path="/opt/rocm/llvm/bin:/opt/rocm/lib/llvm/bin")
    if gxx is None:
        pytest.skip("no host compiler")
    tmp = tmp_path_factory.mktemp("layout")
    src, exe = tmp / "layout.cpp", tmp / "layout"
    src.write_text('#include <cstdio>\n#include "mx4_layout.hpp"\nusing namespace xfc;\n'
                   'int main() {\n  int f; long long a, b, c, d;\n'
                   '  while (scanf("%d %lld %lld %lld %lld", &f, &a, &b, &c, &d) == 5)\n'
                   '    printf("%lld\\n", (long long)(f == 0 ? mx_code_bytes(a) : f == 1 ? mx_scale_bytes(a) : f == 2 ? mx_step_codes(a) : f == 3 ? mx_step_scales(a)\n'
                   '      : f == 4 ? mx_wide(a, b) : f == 5 ? mx_label(a, b) : f == 6 ? mx_tile(a) : f == 7 ? mx_row(a) : f == 8 ? mx_code_at(a, b, c, d) : mx_scale_at(a, b, c)));\n}\n')
    subprocess.run([gxx, "-std=c++17", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    names = ("code_bytes", "scale_bytes", "step_codes", "step_scales", "wide", "label", "tile", "row", "code_at", "scale_at")

    def of(calls):
        text = "\n".join(" ".join(map(str, (names.index(c[0]), *c[1:], *(0,) * (5 - len(c))))) for c in calls)
        return [int(v) for v in subprocess.run([str(exe)], check=True, input=text, stdout=subprocess.PIPE, text=True).stdout.split()]

    return of


@pytest.mark.parametrize("d", [8, 128, 768, (1 << 26) - 8, (1 << 26) + 8, (1 << 26) + 136, 1 << 27, (1 << 30) + 40, (1 << 31) - 128])
def test_steps_of_any_width_lie_in_their_unit(layout, d):
    """The last step's codes and scales end where the unit's do, as quantising takes widths up to 2^31 - 128 dims."""
    last, blocks = -(-d // 128) - 1, -(-d // 32)
    codes, scales, at, scale_at, wide = layout([("code_bytes", d), ("scale_bytes", d), ("step_codes", last), ("step_scales", last), ("wide", last, blocks)])
    assert codes == 1024 * blocks and scales == 256 * (last + 1)
    assert wide == blocks - 4 * last and at == 4096 * last and at + 64 * 16 * wide == codes
    assert scale_at == 256 * last and scale_at + 256 == scales


@pytest.mark.parametrize("d", [8, 96, 128, 200, 768])
def test_blocks_of_a_unit_fill_it_once(layout, d):
    blocks = -(-d // 32)
    place = layout([(f, label) for label in range(64) for f in ("tile", "row")])
    place = list(zip(place[0::2], place[1::2]))
    assert layout([("label", t, r) for t, r in place]) == list(range(64))
    assert sorted(layout([("code_at", t, r, b, blocks) for t, r in place for b in range(blocks)])) == list(range(0, 1024 * blocks, 16))
    scales = layout([("scale_at", t, r, b) for t, r in place for b in range(blocks)])
    assert len(set(scales)) == 64 * blocks and min(scales) >= 0 and max(scales) < 256 * -(-d // 128)


@pytest.mark.parametrize("d", [4096, 9088, 16384])
def test_the_last_block_of_what_products_and_pairs_take(layout, d):
    blocks = d // 32
    at, scale = layout([("code_at", 3, 15, blocks - 1, blocks), ("scale_at", 3, 15, blocks - 1)])
    assert at + 16 == 1024 * blocks and 0 < scale < 256 * -(-d // 128)
