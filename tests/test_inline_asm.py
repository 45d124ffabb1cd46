"""Inline assembly of the kernels names the registers it writes: a statement that sets m0 has it among its clobbers, so that the
compiler keeps no value of its own there.  CPU only."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'treeattn_amd', 'csrc')


def statements(text):
    """The arguments of every asm statement."""
    for m in re.finditer(r'\basm\s+(?:volatile\s*)?\(', text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != '\\':
                quoted = not quoted
            elif not quoted:
                depth += (c == '(') - (c == ')')
            i += 1
        yield text[m.end():i - 1]


def test_m0_is_named_where_it_is_written():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, '*.h*'))):
        for s in statements(open(path).read()):
            if re.search(r's_mov_b32 m0\b', s):
                seen += 1
                assert re.search(r'"m0"', s), (os.path.basename(path), s)
    assert seen >= 3
