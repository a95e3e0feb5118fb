"""Inline assembly names every register that it writes outside of its operands: the compiler may keep values there otherwise."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "elf_amd", "csrc")


def _statements():
	for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
		with open(path) as f:
			text = re.sub(r"//[^\n]*", "", f.read())
		for m in re.finditer(r"\basm\s+volatile\s*\(", text):
			depth, i, quoted = 1, m.end(), False
			while depth:
				c = text[i]
				if c == '"' and text[i - 1] != "\\":
					quoted = not quoted
				elif not quoted:
					depth += (c == "(") - (c == ")")
				i += 1
			yield f"{os.path.basename(path)}: {text[m.start():i]}", text[m.end() : i - 1]


def test_m0_and_scc_are_named():
	seen = 0
	for where, body in _statements():
		strings = re.findall(r'"((?:[^"\\]|\\.)*)"', body)
		template, rest = strings[0], strings[1:]
		for op in re.split(r"\\n\\t|\\n", template):
			op = op.strip()
			if re.match(r"s_\w+ m0\b", op):
				seen += 1
				assert "m0" in rest, where
			if re.match(r"s_(add|sub|and|or|xor|lshl|lshr|cmp)\w*_[ub]\w*32\b", op):
				assert "scc" in rest, where
	assert seen >= 4
