#!/bin/bash
# Build libpss.so of another commit into build/ab/<name>/ (same-box A/B through PSS_LIB), by that
# commit's own makefile:
#   bash tools/build_ref_variant.sh <name> <git-ref> [-DFLAG ...]
# Commits from before the makefile switched packed fp32 arithmetic off get that switch, too: their
# kernels are then not quite what they were, but some forms of it are not reliable on this hardware.
set -e
cd "$(dirname "$0")/.."
name=$1; ref=$2; shift 2
O=$PWD/build/ab/$name; rm -rf "$O"; mkdir -p "$O/src"
git archive "$ref" partiallyshuffledistributedsampler_amd/csrc include | tar -x -C "$O/src"
make -s -j8 -C "$O/src/partiallyshuffledistributedsampler_amd/csrc" OUT="$O/libpss.so" OBJDIR="$O/obj" \
  CXXFLAGS="-O3 -std=c++17 -fPIC -Wall -Wno-unused-result -Xclang -target-feature -Xclang -packed-fp32-ops $*" "$O/libpss.so"
# (a shared library links with symbols missing; loading it finds them)
python3 -c "import ctypes, sys; ctypes.CDLL(sys.argv[1])" "$O/libpss.so"
rm -rf "$O/obj" "$O/src"
echo "built build/ab/$name/libpss.so"
