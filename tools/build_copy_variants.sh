#!/bin/bash
# Diagnostic builds of libfedcodec for the copy-kernel A/B (FC_COPY_U loads in flight
# per lane, FC_COPY_NT non-temporal, FC_COPY_WG workgroups per CU).
set -e
cd "$(dirname "$0")/.."
python3 -m federated_amd.build cpu8=FC_COPY_U=8 cpnt=FC_COPY_NT=1 cpu8nt=FC_COPY_U=8,FC_COPY_NT=1 cpu2=FC_COPY_U=2,FC_COPY_WG=16
